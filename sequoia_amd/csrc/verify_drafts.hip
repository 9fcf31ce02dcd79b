// Verification of the drafted tokens of a batch, from given uniforms.  Sequence b drafted n tokens d_0 .. d_{n-1}; with the
// target's rows p_0 .. p_n and the draft's q_0 .. q_{n-1} (softmax of logits / T), d_i is accepted while u_i q_i(d_i) < p_i(d_i);
// the token that follows is drawn from max(p_k - q_k, 0) at the first rejection k, from p_n behind the last accepted one: the
// first token whose running mass exceeds u * total.  T = 0: p is its first maximum.
//
// Every outcome is a comparison, so everything that one rests on is 64-bit: the sums of exponentials, the two probabilities and
// the running mass (an fp32 sum of a vocabulary's exponentials is off by 1e-7 or so, next to a border per 1e-5: one draw in a
// thousand would differ from the definition's).  Three launches: per part of a row the maximum and the sum; per part
// and sequence the accept walk (redundant in every part) and the part's residual mass; per sequence the part that holds the draw
// and the token in it.  The first reads every logit once; the others touch two rows a sequence and are bound by latency.  (The
// draw in the second launch's last workgroup of a sequence: every workgroup's release writes its XCD's L2 back, and the 21 us of
// the two launches at 64 sequences of 32000 tokens became 28.)
// One sequence of five drafted tokens, 32000 tokens, fp16: 17.6 us (4.4 + 5.7 + 7.8 of the launches, each a chain of loads).  64
// sequences of 0-8: 38.8 us, 20 of it the first launch, bound by its 64-bit operations (5.3 cycles a wave's instruction here) and
// not by the 5.2 TB/s that its bytes would allow; 24 sequences of 2-6 with 128261 tokens, bf16: 48.8 us.
#include "paged.h"

#define VD_THREADS 256
// the walk and the draw: eight waves (a drafted token each), four tokens a lane
#define VD_DRAW_THREADS 512
#define VD_DRAW_PART 2048

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
    int n_seqs, n_drafts, vocab, parts, draw_parts;
    RowPart* stats;          // [n_drafts + n_seqs target rows | n_drafts draft rows][parts]
    double* mass;            // [n_seqs][draw_parts][2]: residual, p itself
    Decided* decided;        // [n_seqs]
    float* token_logit;      // [rows of stats]: the logit of the drafted token that the row judges, or was drawn from
};

// log2(e) / T; 0: greedy.  1e30 is as flat as any temperature above it
__device__ __forceinline__ double log2e_over(float t) {
    return t > 0.f ? 1.4426950408889634 / (double)(t < 1e30f ? t : 1e30f) : 0.0;
}
// e^((x - top) / T) with c = log2(e) / T, x <= top: 2^t, t = (x - top) c, to 4e-14 (NaN stays).  t = k + f, |f| <= 1/2, and
// 2^f = 1 + f g(f) with g of degree 8, interpolated at the Chebyshev nodes; the weight of the maximum is exactly 1.  t stops at
// -1080, where the result is 0.
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
// The sum of eight of them beside a sum that holds a 1 already, in two thirds of the instructions (they bound the first launch): t
// by one fused operation from shift = -top c, whose rounding is one factor for the whole sum; a stop at -1020, which no sum beside
// a 1 notices, so that k goes straight into the exponent's bits.  Four at a time: one alone is a chain of dependent instructions.
// Not for NaN.
__device__ __forceinline__ double weights_in_sum(const Exp2& E, const float (&x)[8], double shift, double c) {
    const double big = 6755399441055744.0;
    double sum = 0.0;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
        double f[4], g[4];
        uint32_t k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_fmax(__builtin_fma((double)x[h + j], c, shift), -1020.0);
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

// N consecutive logits from `at`; -inf behind `end`.  Rows of an odd vocabulary start at any element: the 16-byte loads need no
// alignment on this hardware, and the compiler is told of none.
template <typename T, int N> __device__ __forceinline__ void load_row(const T* row, int at, int end, float (&x)[N]) {
    if (at + N <= end) {
        T v[N];
        __builtin_memcpy(v, row + at, sizeof(v));
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = at + j < end ? (float)row[at + j] : -INFINITY;
    }
}

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

template <typename T, int CHUNKS>
__global__ void __launch_bounds__(VD_THREADS) verify_drafts_stats_kernel(VerifyDraftsParams P) {
    constexpr int PART = 8 * CHUNKS * VD_THREADS;
    __shared__ float s_max[4];
    __shared__ int s_first;
    __shared__ double s_sum[4];
    const int part = blockIdx.x % P.parts, row = blockIdx.x / P.parts, n_target = P.n_drafts + P.n_seqs, lane = threadIdx.x & 63;
    const bool is_t = row < n_target;
    const T* src = is_t ? (const T*)P.target + (int64_t)row * P.ld_t : (const T*)P.draft + (int64_t)(row - n_target) * P.ld_d;
    const int lo = part * PART, hi = lo + PART < P.vocab ? lo + PART : P.vocab;
    float x[CHUNKS][8];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) load_row(src, lo + i * (8 * VD_THREADS) + 8 * threadIdx.x, hi, x[i]);
    // target rows of sequence b end at cu[b + 1] + b + 1, draft rows at cu[b + 1]
    int seq = P.n_seqs;
    for (int base = 0; base < P.n_seqs && seq == P.n_seqs; base += 64) {
        const int i = base + lane;
        const uint64_t hit = __ballot(i < P.n_seqs && (is_t ? P.cu[i + 1] + i + 1 > row : P.cu[i + 1] > row - n_target));
        if (hit) seq = base + __builtin_ctzll(hit);
    }
    if (seq >= P.n_seqs) return;                             // behind the last sequence
    const double c = log2e_over(P.temps ? P.temps[seq] : P.temp);
    // the row's drafted token, if it is in this part: its logit goes to the walk (loaded here, stored at the end)
    const int i_tok = is_t ? row - seq : row - n_target;
    const bool judged = threadIdx.x == 0 && i_tok < P.cu[seq + 1] && i_tok < P.n_drafts;
    float token_logit = 0.f;
    bool mine = false;
    if (judged) {
        const int64_t tok = P.tokens[i_tok];
        mine = tok >= lo && tok < hi;
        if (mine) token_logit = (float)src[tok];
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, x[i][j]);
    const float top = block_max_f32<4>(m, s_max);
    const Exp2 E;
    double sum = 0.0;
    int first = 0x7fffffff;
    bool nan = top == INFINITY;                              // such a row is no distribution either
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) nan |= x[i][j] != x[i][j];
    if (c > 0.0) {
        if (top > -INFINITY) {                               // else nothing in this part counts
            const double shift = -(double)top * c;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) sum += weights_in_sum(E, x[i], shift, c);
        }
    } else if (top > -INFINITY) {                            // greedy: the first maximum
        if (threadIdx.x == 0) s_first = 0x7fffffff;
        __syncthreads();
#pragma unroll
        for (int i = CHUNKS - 1; i >= 0; --i)
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (x[i][j] == top) first = lo + i * (8 * VD_THREADS) + 8 * threadIdx.x + j;
        if (first != 0x7fffffff) atomicMin(&s_first, first);    // a minimum: the order does not matter
        __syncthreads();
        first = s_first;
    }
    sum = wave_sum_f64(nan ? NAN : sum);
    if (lane == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (mine) P.token_logit[row] = token_logit;
    if (threadIdx.x == 0) P.stats[(size_t)row * P.parts + part] = RowPart{top, first, (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3])};
}

// A row's maximum, and the sum of exponentials relative to it, by a group of G lanes (a power of two, no fewer than the parts, at
// most 64: several rows a wave); greedy: the first index of the maximum too.
__device__ __forceinline__ RowTotal row_total(const Exp2& E, const VerifyDraftsParams& P, int row, double c, int G) {
    const RowPart* s = P.stats + (size_t)row * P.parts;
    const int sub = threadIdx.x & (G - 1);
    RowPart mine = sub < P.parts ? s[sub] : RowPart{-INFINITY, 0x7fffffff, 0.0};
    float top = mine.top;
    for (int p = sub + 64; p < P.parts; p += 64) top = fmaxf(top, s[p].top);       // (more than 64 parts: G = 64)
    for (int o = 1; o < G; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    double z = mine.top == -INFINITY ? mine.sum : mine.sum * weight(E, (double)mine.top, (double)top, c);
    int f = mine.top == top ? mine.first : 0x7fffffff;
    for (int p = sub + 64; p < P.parts; p += 64) {
        mine = s[p];
        z += mine.top == -INFINITY ? mine.sum : mine.sum * weight(E, (double)mine.top, (double)top, c);
        if (mine.top == top) f = f < mine.first ? f : mine.first;
    }
    for (int o = 1; o < G; o <<= 1) z += __shfl_xor(z, o, 64);
    if (c == 0.0)
        for (int o = 1; o < G; o <<= 1) { const int w = __shfl_xor(f, o, 64); f = f < w ? f : w; }
    return RowTotal{top, z, f};
}

// Of 4 consecutive tokens: p, and max(p - q, 0), each up to a factor of its own (the rows' sums are multiplied crosswise, not
// divided by: a draw needs no scale)
template <typename T>
__device__ __forceinline__ void residual4(const Exp2& E, const VerifyDraftsParams& P, int b, int at0, const Decided& W, double c, int at, int hi,
                                          double (&p)[4], double (&r)[4]) {
    float x[4], y[4];
    load_row((const T*)P.target + (int64_t)(at0 + b + W.k) * P.ld_t, at, hi, x);
    if (W.two) load_row((const T*)P.draft + (int64_t)(at0 + W.k) * P.ld_d, at, hi, y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[j] = at + j < hi ? weight(E, (double)x[j], W.p_top, c) : 0.0;
        r[j] = p[j];
        if (W.two) {
            const double d = p[j] * W.q_sum - (at + j < hi ? weight(E, (double)y[j], W.q_top, c) * W.p_sum : 0.0);
            r[j] = d < 0.0 ? 0.0 : d;                        // NaN stays
        }
    }
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

// One workgroup a (sequence, part).  All of them judge the sequence's drafted tokens, VD_KEEP at a time (groups of lanes total the
// rows, then a lane a token decides): the first rejection decides which two rows the part's masses are taken from.
#define VD_KEEP 64
template <typename T>
__global__ void __launch_bounds__(VD_DRAW_THREADS) verify_drafts_walk_kernel(VerifyDraftsParams P) {
    constexpr int NW = VD_DRAW_THREADS / 64;
    __shared__ int s_reject;
    __shared__ RowTotal s_tot[2 * VD_KEEP];                  // target rows, draft rows
    __shared__ double s_sum[2][NW];
    const int part = blockIdx.x % P.draw_parts, b = blockIdx.x / P.draw_parts, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int n_target = P.n_drafts + P.n_seqs, at0 = P.cu[b], n = P.cu[b + 1] - at0;
    const double c = log2e_over(P.temps ? P.temps[b] : P.temp);
    const bool greedy = c == 0.0;
    if (at0 < 0 || n < 0 || at0 + n > P.n_drafts) {          // offsets that name no rows
        if (part == 0 && threadIdx.x == 0) { P.accepted[b] = 0; P.next[b] = -1; P.decided[b].draw = 0; }
        return;
    }
    const Exp2 E;
    int G = 1;
    while (G < 64 && G < P.parts) G <<= 1;
    if (threadIdx.x == 0) s_reject = n;
    int base = 0;
    for (;; base += VD_KEEP) {                               // row n follows the last token: nothing to judge there
        const int cnt = n + 1 - base < VD_KEEP ? n + 1 - base : VD_KEEP;
        const bool judge = threadIdx.x < cnt && base + (int)threadIdx.x < n;
        int64_t tok = 0;
        float x = 0.f, y = 0.f, u = 0.f;
        if (judge) {
            const int d = at0 + base + threadIdx.x;
            tok = P.tokens[d]; x = P.token_logit[d + b]; y = P.token_logit[n_target + d]; u = P.u_accept[d];
        }
        const int rows = greedy ? cnt : 2 * cnt;
        for (int j0 = wave * (64 / G); j0 < rows; j0 += NW * (64 / G)) {       // uniform over the wave: its lanes exchange
            const int j = j0 + lane / G, i = base + (j < cnt ? j : j - cnt);
            const bool any = j < cnt || (j < rows && i < n);
            const RowTotal t = row_total(E, P, any ? (j < cnt ? at0 + b + i : n_target + at0 + i) : at0 + b, c, G);
            if (any && (lane & (G - 1)) == 0) s_tot[j < cnt ? j : VD_KEEP + j - cnt] = t;
        }
        __syncthreads();
        if (judge) {
            const RowTotal p = s_tot[threadIdx.x], q = s_tot[VD_KEEP + threadIdx.x];
            bool ok = false;
            if (tok >= 0 && tok < P.vocab) {
                if (greedy) ok = p.sum == 0.0 && p.first == tok;     // first: no index where nothing is above -inf
                else ok = (double)u * weight(E, (double)y, q.top, c) * p.sum < weight(E, (double)x, p.top, c) * q.sum;
            }
            if (!ok) atomicMin(&s_reject, base + (int)threadIdx.x);  // a minimum: the order does not matter
        }
        __syncthreads();
        if (s_reject < base + cnt || base + cnt > n) break;
    }
    const int k = s_reject;
    const bool two = k < n && !greedy;
    const RowTotal p = s_tot[k - base], q = two ? s_tot[VD_KEEP + k - base] : RowTotal{0.0, 1.0, 0};
    const Decided W{k, greedy ? 0 : 1, two ? 1 : 0, p.top, p.sum, q.top, q.sum};
    if (part == 0 && threadIdx.x == 0) {
        P.accepted[b] = k;
        P.decided[b] = W;
        if (greedy) P.next[b] = p.top > -INFINITY && p.sum == 0.0 ? p.first : -1;
    }
    if (greedy) return;

    const int lo = part * VD_DRAW_PART, hi = lo + VD_DRAW_PART < P.vocab ? lo + VD_DRAW_PART : P.vocab;
    double pp[4], rr[4];
    residual4<T>(E, P, b, at0, W, c, lo + 4 * threadIdx.x, hi, pp, rr);
    const double rest = wave_sum_f64((rr[0] + rr[1]) + (rr[2] + rr[3])), all = wave_sum_f64((pp[0] + pp[1]) + (pp[2] + pp[3]));
    if (lane == 0) { s_sum[0][wave] = rest; s_sum[1][wave] = all; }
    __syncthreads();
    if (threadIdx.x < 2) {
        const double* v = s_sum[threadIdx.x];
        P.mass[((size_t)b * P.draw_parts + part) * 2 + threadIdx.x] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
}

// One workgroup a sequence: the part that holds the draw, by every wave for itself, 64 parts at a time; then the token in it.
template <typename T>
__global__ void __launch_bounds__(VD_DRAW_THREADS) verify_drafts_draw_kernel(VerifyDraftsParams P) {
    __shared__ int s_hit, s_last;
    __shared__ double s_sum[VD_DRAW_THREADS / 64];
    const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Decided W = P.decided[b];
    const int at0 = P.cu[b];
    const double c = log2e_over(P.temps ? P.temps[b] : P.temp), u_next = (double)P.u_next[b];
    const double* mass = P.mass + (size_t)b * P.draw_parts * 2;
    if (!W.draw) return;
    if (threadIdx.x == 0) { s_hit = 0x7fffffff; s_last = -1; }
    double total[2] = {0.0, 0.0};
    for (int at = 0; at < P.draw_parts; at += 64) {
        const bool in = at + lane < P.draw_parts;
        total[0] += wave_sum_f64(in ? mass[2 * (at + lane)] : 0.0);
        total[1] += wave_sum_f64(in ? mass[2 * (at + lane) + 1] : 0.0);
    }
    const int which = total[0] == 0.0 ? 1 : 0;               // p nowhere above q: p itself
    const double all = which ? total[1] : total[0];
    if (!(all > 0.0 && all < INFINITY)) {                    // NaN: no distribution to draw from
        if (threadIdx.x == 0) P.next[b] = -1;
        return;
    }
    const double goal = u_next * all;
    int found = -1, last_part = 0;
    double before = 0.0, last_before = 0.0, run = 0.0;       // run: mass of the parts before `at`
    for (int at = 0; at < P.draw_parts && found < 0; at += 64) {
        const double v = at + lane < P.draw_parts ? mass[2 * (at + lane) + which] : 0.0;
        const double upto = run + wave_scan_f64(v), prior = upto - v;
        const uint64_t some = __ballot(v > 0.0), hit = __ballot(v > 0.0 && upto > goal);
        if (hit) { const int j = __builtin_ctzll(hit); found = at + j; before = lane_f64(prior, j); }
        else if (some) { const int j = 63 - __builtin_clzll(some); last_part = at + j; last_before = lane_f64(prior, j); }
        run = lane_f64(upto, 63);
    }
    if (found < 0) { found = last_part; before = last_before; }  // rounding left none: the last one that has mass
    const int lo = found * VD_DRAW_PART + 4 * threadIdx.x, hi = (found + 1) * VD_DRAW_PART < P.vocab ? (found + 1) * VD_DRAW_PART : P.vocab;
    const Exp2 E;
    double pp[4], rr[4], v[4];
    residual4<T>(E, P, b, at0, W, c, lo, hi, pp, rr);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = which ? pp[j] : rr[j];
    const double mine = (v[0] + v[1]) + (v[2] + v[3]), scan = wave_scan_f64(mine);
    if (lane == 63) s_sum[wave] = scan;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += s_sum[w];
    run = before + (scan - mine);
    int hit = 0x7fffffff, last = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        run += v[j];
        if (v[j] > 0.0) {
            last = lo + j;
            if (run > goal && hit == 0x7fffffff) hit = lo + j;
        }
    }
    if (hit != 0x7fffffff) atomicMin(&s_hit, hit);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (threadIdx.x == 0) P.next[b] = s_hit != 0x7fffffff ? s_hit : s_last;     // (likewise)
}

// A statistics workgroup lives about 5 us, nearly all of it waiting for its first loads: with more of them than fit the card at
// once (8 a CU), parts of 4096 tokens cost a second round, so the parts grow to 16384.
static int stats_part(int64_t rows, int vocab) { return rows * ((vocab - 1) / 4096 + 1) > 2048 ? 16384 : 4096; }

struct DraftLayout { size_t mass, decided, token_logit, bytes; int part, parts, draw_parts; };
static DraftLayout draft_layout(int n_seqs, int n_drafts, int vocab) {
    DraftLayout L;
    const size_t rows = (size_t)2 * n_drafts + n_seqs;
    L.part = stats_part((int64_t)rows, vocab);
    L.parts = (vocab - 1) / L.part + 1;
    L.draw_parts = (vocab - 1) / VD_DRAW_PART + 1;
    L.mass = rows * L.parts * sizeof(RowPart);
    L.decided = L.mass + (size_t)n_seqs * L.draw_parts * 2 * sizeof(double);
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
    const int64_t rows = 2 * (int64_t)n_drafts + n_seqs;
    if (rows * L.parts > PAGED_MAX_GRID || (int64_t)n_seqs * L.draw_parts > PAGED_MAX_GRID / 2) return SQ_EUNSUPPORTED;
    char* ws = (char*)workspace;
    VerifyDraftsParams P = {target_logits, draft_logits, ld_target, ld_draft, d_draft_tokens, d_cu_drafts, d_u_accept, d_u_next, d_temperature,
                            temperature, d_n_accepted, d_next_tokens, n_seqs, n_drafts, vocab, L.parts, L.draw_parts, (RowPart*)ws,
                            (double*)(ws + L.mass), (Decided*)(ws + L.decided), (float*)(ws + L.token_logit)};
    hipStream_t st = (hipStream_t)stream;
#define SQ_V(TT) do { \
        if (L.part == 4096) hipLaunchKernelGGL((verify_drafts_stats_kernel<TT, 2>), dim3((unsigned)(rows * L.parts)), dim3(VD_THREADS), 0, st, P); \
        else hipLaunchKernelGGL((verify_drafts_stats_kernel<TT, 8>), dim3((unsigned)(rows * L.parts)), dim3(VD_THREADS), 0, st, P); \
        hipLaunchKernelGGL((verify_drafts_walk_kernel<TT>), dim3((unsigned)(n_seqs * L.draw_parts)), dim3(VD_DRAW_THREADS), 0, st, P); \
        hipLaunchKernelGGL((verify_drafts_draw_kernel<TT>), dim3((unsigned)n_seqs), dim3(VD_DRAW_THREADS), 0, st, P); \
    } while (0)
    if (dtype == SQ_DTYPE_F16) SQ_V(half_t);
    else if (dtype == SQ_DTYPE_BF16) SQ_V(bf16_t);
    else SQ_V(float);
#undef SQ_V
    return sq_check_launch();
}
