// Verification of the drafted tokens of a batch, from given uniforms.  Sequence b drafted n tokens d_0 .. d_{n-1}; with the
// target's rows p_0 .. p_n and the draft's q_0 .. q_{n-1} (softmax of logits / T), d_i is accepted while u_i q_i(d_i) < p_i(d_i);
// the token that follows is drawn from max(p_k - q_k, 0) at the first rejection k, from p_n behind the last accepted one: the
// first token whose running mass exceeds u * total.  T = 0: p is its first maximum.
//
// Every outcome is a comparison, so everything that one rests on is 64-bit: the sums of exponentials, the two probabilities and
// the running mass (an fp32 sum of a vocabulary's exponentials is off by 1e-7 or so, next to a border per 1e-5: one draw in a
// thousand would differ from the definition's).  Three launches: per part of a row the maximum and the sum; per sequence and block of
// tokens the accept walk (redundant in every block) and the block's residual mass; per sequence the block that holds the draw and
// the token in it.  The first reads every logit once; the others touch two rows a sequence and are bound by the latency of their
// chains of loads, so that neither has a barrier.  (The draw in the second launch's last workgroup of a sequence: every workgroup's
// release writes its XCD's L2 back, and the two launches' time grew by a third.)
// One sequence of five drafted tokens, 32000 tokens, fp16: 11.8 us on the device.  64 sequences of 0-8: 31.9 us, 19 of it the first
// launch, bound by the vector ALU -- 21 instructions a logit, of which 17 are 64-bit; every one of them takes four
// cycles and a little, 64-bit or not -- and not by the 5.1 TB/s that its bytes would allow.  24 sequences of 2-6 with 128261 tokens,
// bf16: 43 us, 28 of it the first launch.
#include "paged.h"

#define VD_THREADS 256
// The walk and the draw: tokens a lane, and a wave.  More of them a wave: fewer waves judge the same tokens, and more instructions
// stand between its loads and its end.  4 | 8 | 16: one sequence 11.0 | 11.5 | 13.4 us, 24 sequences of 128261 tokens 45.8 | 42.3 | 43.3.
#define VD_LANE 8
#define VD_BLOCK (64 * VD_LANE)

struct RowPart { float top; int first; double sum; };      // maximum, its first index, sum of exp((x - top) / T)
struct RowTotal { double top, sum; int first; };
// accepted tokens; whether a token is still to be drawn, and from two rows; their maxima and sums
struct Decided { int k, draw, two; double p_top, p_sum, q_top, q_sum; };

struct VerifyDraftsParams {
    const void *target, *draft; int64_t ld_t, ld_d;
    const int64_t* tokens;
    const int32_t* cu;
    const float *u_accept, *u_next, *temps;
    float temp;
    int32_t* accepted; int64_t* next;
    int n_seqs, n_drafts, vocab, parts, blocks;
    int group_shift;         // 1 << group_shift lanes total a row
    RowPart* stats;          // [n_drafts + n_seqs target rows | n_drafts draft rows][parts]
    double* mass;            // [n_seqs][blocks][2]: residual, p itself
    Decided* decided;        // [n_seqs]
    float* token_logit;      // [rows of stats]: the logit of the drafted token that the row judges, or was drawn from
};

// log2(e) / T; 0: greedy.  An infinite T is the largest finite one (0 would be greedy)
__device__ __forceinline__ double log2e_over(float t) {
    return t > 0.f ? 1.4426950408889634 / (double)fminf(t, 0x1.fffffep127f) : 0.0;
}
// e^((x - top) / T) with c = log2(e) / T, x <= top: 2^t, t = (x - top) c, to 4e-14, and |t| 2^-53 from t's own rounding (NaN
// stays).  t = k + f, |f| <= 1/2, and 2^f = 1 + f g(f) with g of degree 8, interpolated at the Chebyshev nodes; the weight of the
// maximum is exactly 1.  t stops at -1080, where the result is 0.
struct Exp2 {
    double g[9];
    __device__ __forceinline__ Exp2()
        : g{1.020121756124497e-07, 1.3255217458568395e-06, 1.5252695957285255e-05, 0.00015403455885944662, 0.0013333558165461892,
            0.009618129159357978, 0.05550410866482476, 0.24022650695813147, 0.6931471805599448} {
        // kept in scalar registers: as literals every one costs two moves in front of its multiply-add
#pragma unroll
        for (int i = 0; i < 9; ++i) asm("" : "+s"(g[i]));
    }
};
__device__ __forceinline__ double exp2_parts(const Exp2& E, double t, uint32_t& k) {       // 2^t = result * 2^k
    const double big = 6755399441055744.0, kb = t + big;     // 1.5 * 2^52: adding it leaves the nearest integer in the low bits
    const double f = t - (kb - big);
    double g = E.g[0];
#pragma unroll
    for (int i = 1; i < 9; ++i) g = __builtin_fma(g, f, E.g[i]);
    k = (uint32_t)__builtin_bit_cast(uint64_t, kb);
    return __builtin_fma(g, f, 1.0);
}
__device__ __forceinline__ double weight(const Exp2& E, double x, double top, double c) {
    double t = (x - top) * c;
    t = t < -1080.0 ? -1080.0 : t;
    uint32_t k;
    const double g = exp2_parts(E, t, k);
    return __builtin_amdgcn_ldexp(g, (int)k);
}
// The sum of eight of them beside a sum that holds a 1 already, in fewer instructions (they bound the first launch): a stop at -1020,
// which no sum beside a 1 notices, so that k goes straight into the exponent's bits.  Four at a time: one alone is a chain of
// dependent instructions.  x - top comes before the factor, as in weight(): x c - top c in one fused operation saves an instruction
// (31.5 | 31.9 us for 64 sequences) but is off by the rounding of top c, which the other side of a comparison does not have: 1e-15 of
// the sum at ordinary temperatures, enough to accept what ties, 2e-7 at T = 1e-8, a factor of 4 at 1e-15, and no number at all below.
// Not for NaN.
__device__ __forceinline__ double weights_in_sum(const Exp2& E, const float (&x)[8], double top, double c) {
    const double big = 6755399441055744.0;
    double sum = 0.0;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
        double f[4], g[4];
        uint32_t k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_fmax(((double)x[h + j] - top) * c, -1020.0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double kb = f[j] + big;
            k[j] = (uint32_t)__builtin_bit_cast(uint64_t, kb);
            f[j] -= kb - big;
            g[j] = E.g[0];
        }
#pragma unroll
        for (int i = 1; i < 9; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = __builtin_fma(g[j], f[j], E.g[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x2 w = __builtin_bit_cast(u32x2, __builtin_fma(g[j], f[j], 1.0));
            w[1] += k[j] << 20;
            g[j] = __builtin_bit_cast(double, w);
        }
        sum += (g[0] + g[1]) + (g[2] + g[3]);
    }
    return sum;
}

// N consecutive logits of a row: tokens [at, at + N), or, where those would pass `end` (uniform, the end of a part or of the row), the
// last N before it; a row of fewer than VD_SHORT tokens is taken apart.  Kept as loaded and without a branch, so that nothing waits
// for them before value() does: a row's loads are all in flight at once.  Rows of an odd vocabulary start at any element: the
// 16-byte loads need no alignment on this hardware, and the compiler is told of none.
#define VD_SHORT 8
static_assert(VD_SHORT >= VD_LANE && VD_SHORT >= 8, "a row that is not taken apart holds a lane's tokens");
template <typename T, int N, bool SHORT> struct Logits {
    uint32_t w[N * sizeof(T) / 4];
    int from;                                                // the first one's token
    __device__ __forceinline__ void load(const T* row, int at, int end) {
        if constexpr (!SHORT) {
            from = at < end - N ? at : end - N;
            __builtin_memcpy(w, row + from, sizeof(w));
        } else {
            from = at;
            T v[N];
            for (int j = 0; j < N; ++j) v[j] = row[at + j < end ? at + j : end - 1];
            __builtin_memcpy(w, v, sizeof(w));
        }
    }
    // not looked at before `v` is there: values are widened where they are used, instead of early, or once and kept
    template <typename V> __device__ __forceinline__ void behind(V& v) {
#pragma unroll
        for (uint32_t& x : w) asm volatile("" : "+v"(x), "+v"(v));
    }
    __device__ __forceinline__ float value(int j) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[j]);
        else return (float)__builtin_bit_cast(T, (uint16_t)(w[j / 2] >> (16 * (j & 1))));
    }
    __device__ __forceinline__ bool counts(int j, int at, int end) const { return from + j >= at && from + j < end; }
};

__device__ __forceinline__ double lane_f64(double v, int lane) {                   // lane: uniform
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {                         // fixed order
#define SQ_STEP(n) { const uint64_t b = __builtin_bit_cast(uint64_t, v); \
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, SQ_DPP_ROW_ROR(n), 0xf, 0xf, false); \
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), SQ_DPP_ROW_ROR(n), 0xf, 0xf, false); \
        v += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo); }
    SQ_STEP(8) SQ_STEP(4) SQ_STEP(2) SQ_STEP(1)
#undef SQ_STEP
    return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}

// (fmaxf() would first make every bf16 value canonical)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// a uniform element, by the scalar unit: its wait is not one for the vector loads in flight
template <typename V> __device__ __forceinline__ V scalar_load(const V* p) {
    return *(const __attribute__((address_space(4))) V*)(uintptr_t)p;
}

template <typename T, int CHUNKS, bool SHORT>
__global__ void __launch_bounds__(VD_THREADS, 6) verify_drafts_stats_kernel(VerifyDraftsParams P) {
    constexpr int PART = 8 * CHUNKS * VD_THREADS;
    __shared__ float s_max[4];
    __shared__ int s_first;
    __shared__ double s_sum[4];
    const int part = blockIdx.x % P.parts, row = blockIdx.x / P.parts, n_target = P.n_drafts + P.n_seqs, lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const bool is_t = row < n_target;
    const T* src = is_t ? (const T*)P.target + (int64_t)row * P.ld_t : (const T*)P.draft + (int64_t)(row - n_target) * P.ld_d;
    const int lo = part * PART, hi = lo + PART < P.vocab ? lo + PART : P.vocab;
    // target rows of sequence b end at cu[b + 1] + b + 1, draft rows at cu[b + 1].  The first 64 ends come before the row: loads end
    // in order, and the chunks of the row are summed as they come
    const int first_end = P.cu[(lane < P.n_seqs ? lane : 0) + 1];
    asm volatile("" ::: "memory");                           // (left alone, the load sinks to its use)
    Logits<T, 8, SHORT> row8[CHUNKS];
    const int at0 = lo + 8 * threadIdx.x;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) row8[i].load(src, at0 + i * (8 * VD_THREADS), hi);
    auto values = [&](int i, float (&x)[8]) {                // -inf where another lane has them, and behind the end
        const int at = at0 + i * (8 * VD_THREADS);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = row8[i].value(j);
        if (__any(at + 8 > hi)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = row8[i].counts(j, at, hi) ? x[j] : -INFINITY;
        }
    };
    auto ends_behind = [&](int i, int end) { return __ballot((i < P.n_seqs) & (end + (is_t ? i + 1 : n_target) > row)); };
    uint64_t hit = ends_behind(lane, first_end);
    int seq = 0;
    if (!hit) {
        for (seq = 64; seq < P.n_seqs; seq += 64) {
            hit = ends_behind(seq + lane, P.cu[(seq + lane < P.n_seqs ? seq + lane : 0) + 1]);
            if (hit) break;
        }
        if (!hit) return;                                    // behind the last sequence
    }
    seq += __builtin_ctzll(hit);
    seq = __builtin_amdgcn_readfirstlane(seq);
    const double c = log2e_over(P.temps ? scalar_load(P.temps + seq) : P.temp);
    // the row's drafted token, if it is in this part: its logit goes to the walk (loaded here, stored at the end)
    const int i_tok = is_t ? row - seq : row - n_target;
    int64_t tok = -1;
    if (i_tok >= 0 && i_tok < scalar_load(P.cu + seq + 1) && i_tok < P.n_drafts) tok = scalar_load(P.tokens + i_tok);
    const bool mine = threadIdx.x == 0 && tok >= lo && tok < hi;
    const T token_logit = src[tok >= lo && tok < hi ? tok : lo];
    // the wave's maximum so far, and its lanes' sums relative to it
    const Exp2 E;
    float top = -INFINITY, best = -INFINITY;
    int first = 0x7fffffff;
    double sum = 0.0;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        float x[8];
        row8[i].behind(sum);
        values(i, x);
        float m = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7]));
#pragma unroll
        for (int j = 0; j < 8; j += 2) nan |= __builtin_isunordered(x[j], x[j + 1]);
        if (c > 0.0) {
            if (__any(m > top)) {                            // (seldom, after a row's first chunks)
                m = wave_max_f32_dpp(m);
                if (top > -INFINITY) sum *= weight(E, (double)top, (double)m, c);
                top = m;
            }
            if (top > -INFINITY) sum += weights_in_sum(E, x, (double)top, c);       // else nothing so far counts
        } else {                                             // greedy: the first maximum
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (x[j] > best) { best = x[j]; first = row8[i].from + j; }
        }
    }
    if (c == 0.0) top = wave_max_f32_dpp(best);
    nan |= top == INFINITY;                                  // such a row is no distribution either
    sum = wave_sum_f64(nan ? NAN : sum);
    if (threadIdx.x == 0) s_first = 0x7fffffff;
    if (lane == 0) { s_max[wave] = top; s_sum[wave] = sum; }
    __syncthreads();
    top = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    if (c == 0.0) {
        if (best == top && best > -INFINITY) atomicMin(&s_first, first);         // a minimum: the order does not matter
        __syncthreads();
    }
    if (mine) P.token_logit[row] = (float)token_logit;
    if (threadIdx.x == 0) {
        double s[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) s[w] = s_max[w] == -INFINITY ? s_sum[w] : s_sum[w] * weight(E, (double)s_max[w], (double)top, c);
        P.stats[(size_t)row * P.parts + part] = RowPart{top, s_first, (s[0] + s[1]) + (s[2] + s[3])};
    }
}

// Maxima of rows, and the sums of exponentials relative to them, N rows at once by a group of G lanes (a power of two, no fewer than
// the parts, at most 64); greedy: the first index of the maximum too.
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false); }
template <int N>
__device__ __forceinline__ void row_totals(const Exp2& E, const VerifyDraftsParams& P, const int (&row)[N], double c, RowTotal (&t)[N]) {
    const int G = 1 << P.group_shift, sub = threadIdx.x & (G - 1);
    RowPart mine[N];
#pragma unroll
    for (int r = 0; r < N; ++r) {
        mine[r] = P.stats[(size_t)row[r] * P.parts + (sub < P.parts ? sub : 0)];
        if (sub >= P.parts) mine[r] = RowPart{-INFINITY, 0x7fffffff, 0.0};
        t[r].top = mine[r].top;
    }
    if (P.parts > 64) {                                      // (then G = 64)
        for (int r = 0; r < N; ++r)
            for (int p = sub + 64; p < P.parts; p += 64) t[r].top = fmax(t[r].top, (double)P.stats[(size_t)row[r] * P.parts + p].top);
    }
    // the lane's value and its partner's, over growing distances of a group: all of its lanes end with the same bits
#define SQ_GROUP(STEP) do { \
        if (G > 1) { STEP(dpp<0xB1>); } if (G > 2) { STEP(dpp<0x4E>); }              /* quad_perm: lanes 1 and 2 apart */ \
        if (G > 4) { STEP(dpp<0x141>); } if (G > 8) { STEP(dpp<0x140>); }            /* row_half_mirror, row_mirror */ \
        if (G > 16) { STEP(SQ_X16); } if (G > 32) { STEP(SQ_X32); } \
    } while (0)
#define SQ_X16(v) __shfl_xor(v, 16, 64)
#define SQ_X32(v) __shfl_xor(v, 32, 64)
#define SQ_MAX(X) for (int r = 0; r < N; ++r) { const float w = __builtin_bit_cast(float, X(__builtin_bit_cast(int, (float)t[r].top))); t[r].top = fmax(t[r].top, (double)w); }
#define SQ_SUM(X) for (int r = 0; r < N; ++r) { const uint64_t z = __builtin_bit_cast(uint64_t, t[r].sum); const uint32_t w0 = X((int)(uint32_t)z), w1 = X((int)(uint32_t)(z >> 32)); \
        t[r].sum += __builtin_bit_cast(double, ((uint64_t)w1 << 32) | w0); }
#define SQ_MIN(X) for (int r = 0; r < N; ++r) { const int w = X(t[r].first); t[r].first = t[r].first < w ? t[r].first : w; }
    SQ_GROUP(SQ_MAX);
#pragma unroll
    for (int r = 0; r < N; ++r) {
        t[r].sum = mine[r].top == -INFINITY ? mine[r].sum : mine[r].sum * weight(E, (double)mine[r].top, t[r].top, c);
        t[r].first = mine[r].top == t[r].top ? mine[r].first : 0x7fffffff;
    }
    if (P.parts > 64) {
        for (int r = 0; r < N; ++r)
            for (int p = sub + 64; p < P.parts; p += 64) {
                const RowPart m = P.stats[(size_t)row[r] * P.parts + p];
                t[r].sum += m.top == -INFINITY ? m.sum : m.sum * weight(E, (double)m.top, t[r].top, c);
                if (m.top == t[r].top) t[r].first = t[r].first < m.first ? t[r].first : m.first;
            }
    }
    SQ_GROUP(SQ_SUM);
    if (c == 0.0) SQ_GROUP(SQ_MIN);
#undef SQ_MIN
#undef SQ_SUM
#undef SQ_MAX
#undef SQ_X32
#undef SQ_X16
#undef SQ_GROUP
}

// Of VD_LANE consecutive tokens from `at` on (of `from` on, near the end): p, and max(p - q, 0), each up to a factor of its own (the rows'
// sums are multiplied crosswise, not divided by: a draw needs no scale)
template <typename T, bool SHORT>
__device__ __forceinline__ int residual4(const Exp2& E, const VerifyDraftsParams& P, int b, int at0, const Decided& W, double c, int at, int hi,
                                         double (&p)[VD_LANE], double (&r)[VD_LANE]) {
    Logits<T, VD_LANE, SHORT> x, y;
    x.load((const T*)P.target + (int64_t)(at0 + b + W.k) * P.ld_t, at, hi);
    // (without a draft's row, the target's once more)
    y.load(W.two ? (const T*)P.draft + (int64_t)(at0 + W.k) * P.ld_d : (const T*)P.target + (int64_t)(at0 + b + W.k) * P.ld_t, at, hi);
#pragma unroll
    for (int j = 0; j < VD_LANE; ++j) {
        const bool in = x.counts(j, at, hi);
        p[j] = in ? weight(E, (double)x.value(j), W.p_top, c) : 0.0;
        r[j] = p[j];
        if (W.two) {
            const double d = p[j] * W.q_sum - (in ? weight(E, (double)y.value(j), W.q_top, c) * W.p_sum : 0.0);
            r[j] = d < 0.0 ? 0.0 : d;                        // NaN stays
        }
    }
    return x.from;
}

__device__ __forceinline__ double sum_of(const double (&v)[VD_LANE]) {
    double s = v[0];
#pragma unroll
    for (int j = 1; j < VD_LANE; ++j) s += v[j];
    return s;
}
// running sums over the lanes
__device__ __forceinline__ double wave_scan_f64(double v) {
    const int lane = threadIdx.x & 63;
#define SQ_STEP(n) { const uint64_t b = __builtin_bit_cast(uint64_t, v);        /* row_shr: the lane n below, of the same 16 */ \
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, 0x110 + (n), 0xf, 0xf, true); \
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), 0x110 + (n), 0xf, 0xf, true); \
        v += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo); }
    SQ_STEP(1) SQ_STEP(2) SQ_STEP(4) SQ_STEP(8)
#undef SQ_STEP
    const double a = lane_f64(v, 15), b = a + lane_f64(v, 31), c = b + lane_f64(v, 47);
    return v + (lane < 16 ? 0.0 : lane < 32 ? a : lane < 48 ? b : c);
}

// One wave a (sequence, block of tokens), all of them for themselves: a barrier costs more than what the waves of a workgroup could
// share.  Groups of G lanes judge a drafted token each, 64 / G at a time: the group totals the token's two rows and decides.  The
// first rejection, or the row behind the last token, decides which two rows the block's masses are taken from.
template <typename T, bool SHORT>
__global__ void __launch_bounds__(VD_THREADS) verify_drafts_walk_kernel(VerifyDraftsParams P) {
    const int item = __builtin_amdgcn_readfirstlane(blockIdx.x * (VD_THREADS / 64) + threadIdx.x / 64), lane = threadIdx.x & 63;
    const int b = item / P.blocks, block = item - b * P.blocks;
    if (b >= P.n_seqs) return;
    const int n_target = P.n_drafts + P.n_seqs, at0 = P.cu[b], n = P.cu[b + 1] - at0;
    const double c = log2e_over(P.temps ? P.temps[b] : P.temp);
    const bool greedy = c == 0.0;
    if (at0 < 0 || n < 0 || at0 + n > P.n_drafts) {          // offsets that name no rows
        if (block == 0 && lane == 0) { P.accepted[b] = 0; P.next[b] = -1; P.decided[b].draw = 0; }
        return;
    }
    if (greedy && block) return;
    const Exp2 E;
    RowTotal t[2];                                           // of the target's row, of the draft's
    int k, from;                                             // from: the lane whose group totalled the deciding rows
    for (int base = 0;; base += 64 >> P.group_shift) {
        const int j = base + (lane >> P.group_shift), i = j < n ? j : n;         // row n follows the last token: nothing to judge there
        const int d = at0 + (i < n ? i : n - 1);
        const int row[2] = {at0 + b + i, n ? n_target + d : at0 + b};    // (no tokens: there may be no draft's row at all)
        int64_t tok = -1;
        float x = 0.f, y = 0.f, u = 0.f;
        if (n) { tok = P.tokens[d]; x = P.token_logit[d + b]; y = P.token_logit[n_target + d]; u = P.u_accept[d]; }
        row_totals(E, P, row, c, t);
        bool ok;
        if (greedy) ok = t[0].sum == 0.0 && t[0].first == tok;           // first: no index where nothing is above -inf
        else ok = (double)u * weight(E, (double)y, t[1].top, c) * t[0].sum < weight(E, (double)x, t[0].top, c) * t[1].sum;
        ok = ok && i < n && tok >= 0 && tok < P.vocab;
        const uint64_t stop = __ballot(!ok);
        if (stop) {                                          // (row n stops it)
            from = __builtin_ctzll(stop);
            k = base + (from >> P.group_shift);
            break;
        }
    }
    const bool two = k < n && !greedy;
    const Decided W{k, greedy ? 0 : 1, two ? 1 : 0, lane_f64(t[0].top, from), lane_f64(t[0].sum, from), lane_f64(t[1].top, from), lane_f64(t[1].sum, from)};
    if (block == 0 && lane == from) {
        P.accepted[b] = k;
        P.decided[b] = W;
        if (greedy) P.next[b] = t[0].top > -INFINITY && t[0].sum == 0.0 ? t[0].first : -1;
    }
    if (greedy) return;

    const int lo = block * VD_BLOCK, hi = lo + VD_BLOCK < P.vocab ? lo + VD_BLOCK : P.vocab;
    double pp[VD_LANE], rr[VD_LANE];
    residual4<T, SHORT>(E, P, b, at0, W, c, lo + VD_LANE * lane, hi, pp, rr);
    const double rest = wave_sum_f64(sum_of(rr)), all = wave_sum_f64(sum_of(pp));
    if (lane < 2) P.mass[((size_t)b * P.blocks + block) * 2 + lane] = lane ? all : rest;
}

// One wave a sequence: the block that holds the draw (a lane sums a run of blocks, the lanes' sums are scanned, then the run that
// holds it is), and the token in it.
template <typename T, bool SHORT>
__global__ void __launch_bounds__(64) verify_drafts_draw_kernel(VerifyDraftsParams P) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const Decided W = P.decided[b];
    const int at0 = P.cu[b];
    const double c = log2e_over(P.temps ? P.temps[b] : P.temp), u_next = (double)P.u_next[b];
    const double* mass = P.mass + (size_t)b * P.blocks * 2;
    const int run = (P.blocks + 63) / 64, first = lane * run, end = first + run < P.blocks ? first + run : P.blocks;
    auto each = [&](auto f) {                                // eight loads at once
        for (int i = 0; i < run; i += 8) {
            double m[8][2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = first + i + j < end ? first + i + j : 0;
                m[j][0] = mass[2 * at]; m[j][1] = mass[2 * at + 1];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (first + i + j < end) f(first + i + j, m[j]);
        }
    };
    double v[2] = {0.0, 0.0};
    each([&](int, const double (&m)[2]) { v[0] += m[0]; v[1] += m[1]; });
    if (!W.draw) return;
    const double rest = wave_scan_f64(v[0]), whole = wave_scan_f64(v[1]);
    const int which = lane_f64(rest, 63) == 0.0 ? 1 : 0;     // p nowhere above q: p itself
    const double mine = which ? v[1] : v[0], upto = which ? whole : rest, all = lane_f64(upto, 63);
    if (!(all > 0.0 && all < INFINITY)) {                    // NaN: no distribution to draw from
        if (lane == 0) P.next[b] = -1;
        return;
    }
    const double goal = u_next * all;
    // where rounding leaves no place whose running mass exceeds the goal, it is the last one that has mass: here and below
    const uint64_t some = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && upto > goal);
    const int owner = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
    double sum = upto - mine, before = 0.0;
    int block = 0;
    bool over = false;
    each([&](int i, const double (&m)[2]) {
        const double one = which ? m[1] : m[0];
        if (one > 0.0 && !over) { block = i; before = sum; over = sum + one > goal; }
        sum += one;
    });
    block = __builtin_amdgcn_readlane(block, owner);
    before = lane_f64(before, owner);

    const int lo = block * VD_BLOCK, hi = lo + VD_BLOCK < P.vocab ? lo + VD_BLOCK : P.vocab;
    const Exp2 E;
    double pp[VD_LANE], rr[VD_LANE], w[VD_LANE];
    const int token = residual4<T, SHORT>(E, P, b, at0, W, c, lo + VD_LANE * lane, hi, pp, rr);
#pragma unroll
    for (int j = 0; j < VD_LANE; ++j) w[j] = which ? pp[j] : rr[j];
    const double own = sum_of(w);
    sum = before + (wave_scan_f64(own) - own);
    int found = -1, behind = -1;                             // first above the goal, last that has mass
#pragma unroll
    for (int j = 0; j < VD_LANE; ++j) {
        sum += w[j];
        if (w[j] > 0.0) {
            behind = token + j;
            if (found < 0 && sum > goal) found = behind;
        }
    }
    const uint64_t f = __ballot(found >= 0), l = __ballot(behind >= 0);
    const int t = f ? __builtin_amdgcn_readlane(found, __builtin_ctzll(f)) : __builtin_amdgcn_readlane(behind, 63 - __builtin_clzll(l | 1));
    if (lane == 0) P.next[b] = t;
}

// Parts of 4096 tokens where the workgroups fit the card at once (8 a CU): a workgroup lives 3 us, most of it waiting for its loads.
// Beyond that parts of 8192, whose chunks are summed while the later ones come.  4096 | 8192 | 16384, 64 sequences of 32000 tokens:
// 19.4 | 18.8 | 20.2 us, 24 of 128261: 30.2 | 28.7 | 28.0.
static int stats_part(int64_t rows, int vocab) { return rows * ((vocab - 1) / 4096 + 1) > 2048 ? 8192 : 4096; }

struct DraftLayout { size_t mass, decided, token_logit, bytes; int part, parts, blocks; };
static DraftLayout draft_layout(int n_seqs, int n_drafts, int vocab) {
    DraftLayout L;
    const size_t rows = (size_t)2 * n_drafts + n_seqs;
    L.part = stats_part((int64_t)rows, vocab);
    L.parts = (vocab - 1) / L.part + 1;
    L.blocks = (vocab - 1) / VD_BLOCK + 1;
    L.mass = rows * L.parts * sizeof(RowPart);
    L.decided = L.mass + (size_t)n_seqs * L.blocks * 2 * sizeof(double);
    L.token_logit = L.decided + (size_t)n_seqs * sizeof(Decided);
    L.bytes = L.token_logit + (rows * sizeof(float) + 15) / 16 * 16;
    return L;
}

extern "C" size_t sq_verify_drafts_workspace_bytes(int n_seqs, int n_drafts, int vocab) {
    if (n_seqs <= 0 || n_drafts < 0 || vocab <= 0) return 0;
    return draft_layout(n_seqs, n_drafts, vocab).bytes;
}

extern "C" int sq_verify_drafts(const void* target_logits, int64_t ld_target, const void* draft_logits, int64_t ld_draft,
                                const int64_t* d_draft_tokens, const int32_t* d_cu_drafts, int n_seqs, int n_drafts, int vocab,
                                const float* d_u_accept, const float* d_u_next, const float* d_temperature, float temperature,
                                int32_t* d_n_accepted, int64_t* d_next_tokens, int dtype, void* workspace, size_t workspace_bytes,
                                void* stream) {
    if (n_seqs < 0 || n_drafts < 0 || vocab <= 0) return SQ_EINVAL;
    if (dtype != SQ_DTYPE_F16 && dtype != SQ_DTYPE_BF16 && dtype != SQ_DTYPE_F32) return SQ_EUNSUPPORTED;
    if (vocab > 1 << 30) return SQ_EUNSUPPORTED;            // tokens are counted in 32 bits, a part past the end
    if (n_seqs == 0) return SQ_OK;
    if (!target_logits || !d_cu_drafts || !d_u_next || !d_n_accepted || !d_next_tokens || ld_target < vocab) return SQ_EINVAL;
    if (n_drafts && (!draft_logits || !d_draft_tokens || !d_u_accept || ld_draft < vocab)) return SQ_EINVAL;
    if (!d_temperature && !(temperature >= 0.f && temperature < INFINITY)) return SQ_EINVAL;
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < sq_verify_drafts_workspace_bytes(n_seqs, n_drafts, vocab)) return SQ_EINVAL;
    const DraftLayout L = draft_layout(n_seqs, n_drafts, vocab);
    const int64_t rows = 2 * (int64_t)n_drafts + n_seqs, walk = ((int64_t)n_seqs * L.blocks + VD_THREADS / 64 - 1) / (VD_THREADS / 64);
    if (rows * L.parts > PAGED_MAX_GRID || (int64_t)n_seqs * L.blocks > PAGED_MAX_GRID / 2) return SQ_EUNSUPPORTED;
    char* ws = (char*)workspace;
    int group_shift = 0;
    while (group_shift < 6 && 1 << group_shift < L.parts) ++group_shift;
    VerifyDraftsParams P = {target_logits, draft_logits, ld_target, ld_draft, d_draft_tokens, d_cu_drafts, d_u_accept, d_u_next, d_temperature,
                            temperature, d_n_accepted, d_next_tokens, n_seqs, n_drafts, vocab, L.parts, L.blocks, group_shift, (RowPart*)ws,
                            (double*)(ws + L.mass), (Decided*)(ws + L.decided), (float*)(ws + L.token_logit)};
    hipStream_t st = (hipStream_t)stream;
#define SQ_V(TT, SS) do { \
        if (L.part == 4096) hipLaunchKernelGGL((verify_drafts_stats_kernel<TT, 2, SS>), dim3((unsigned)(rows * L.parts)), dim3(VD_THREADS), 0, st, P); \
        else hipLaunchKernelGGL((verify_drafts_stats_kernel<TT, 4, SS>), dim3((unsigned)(rows * L.parts)), dim3(VD_THREADS), 0, st, P); \
        hipLaunchKernelGGL((verify_drafts_walk_kernel<TT, SS>), dim3((unsigned)walk), dim3(VD_THREADS), 0, st, P); \
        hipLaunchKernelGGL((verify_drafts_draw_kernel<TT, SS>), dim3((unsigned)n_seqs), dim3(64), 0, st, P); \
    } while (0)
#define SQ_VS(TT) do { if (vocab < VD_SHORT) SQ_V(TT, true); else SQ_V(TT, false); } while (0)
    if (dtype == SQ_DTYPE_F16) SQ_VS(half_t);
    else if (dtype == SQ_DTYPE_BF16) SQ_VS(bf16_t);
    else SQ_VS(float);
#undef SQ_VS
#undef SQ_V
    return sq_check_launch();
}
