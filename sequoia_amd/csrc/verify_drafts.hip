// Verification of the drafted tokens of a batch, from given uniforms.  Sequence b drafted n tokens d_0 .. d_{n-1}; with the
// target's rows p_0 .. p_n and the draft's q_0 .. q_{n-1} (softmax of logits / T), d_i is accepted while u_i q_i(d_i) < p_i(d_i);
// the token that follows is drawn from max(p_k - q_k, 0) at the first rejection k, from p_n behind the last accepted one: the
// first token whose running mass exceeds u * total.  T = 0: p is its first maximum.
//
// Every outcome is a comparison, so everything that one rests on is 64-bit: the sums of exponentials, the two probabilities and
// the running mass (an fp32 sum of a vocabulary's exponentials is off by 1e-7 or so, next to a border per 1e-5: one draw in a
// thousand would differ from the definition's).  Three launches: per 4096-token part and row the maximum and the sum; per part
// and sequence the accept walk (redundant in every part) and the part's residual mass; per sequence the part that holds the draw
// and the token in it.  The first is bound by the bytes of the logits, which it reads once; the others touch two rows a sequence.
#include "paged.h"

#define VD_THREADS 256
#define VD_EPT 16
#define VD_PART (VD_THREADS * VD_EPT)

struct RowPart { float top; int first; double sum; };      // maximum, its first index, sum of exp((x - top) / T)

struct VerifyDraftsParams {
    const void *target, *draft; int64_t ld_t, ld_d;
    const int64_t* tokens;
    const int32_t* cu;
    const float *u_accept, *u_next, *temps;
    float temp;
    int32_t* accepted; int64_t* next;
    int n_seqs, n_drafts, vocab, parts;
    RowPart* stats;          // [n_drafts + n_seqs target rows | n_drafts draft rows][parts]
    double* mass;            // [n_seqs][parts][2]: residual, p itself
};

// e^y for y <= 0 (and NaN) to about 1e-16: y = k ln 2 + r, |r| <= 0.35, Taylor to r^13 / 13!
__device__ __forceinline__ double exp64(double y) {
    y = y < -800.0 ? -800.0 : y;
    const double k = __builtin_rint(y * 1.4426950408889634);
    double r = __builtin_fma(k, -0.6931471824645996, y);            // ln 2 = its fp32 value, k times which is exact, and what is left of it
    r = __builtin_fma(k, 1.904654299957768e-09, r);
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)k);
}

// 8 consecutive logits from `at`; -inf behind `end`.  Rows of an odd vocabulary start at any element: the 16-byte loads need no
// alignment on this hardware, and the compiler is told of none.
template <typename T> __device__ __forceinline__ void load8(const T* row, int at, int end, float (&x)[8]) {
    if (at + 8 <= end) {
        T v[8];
        __builtin_memcpy(v, row + at, sizeof(v));
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = at + j < end ? (float)row[at + j] : -INFINITY;
    }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ double block_sum_f64(double v, double* scratch) {       // 4 waves, fixed order
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

template <typename T>
__global__ void __launch_bounds__(VD_THREADS) verify_drafts_stats_kernel(VerifyDraftsParams P) {
    __shared__ float s_max[4];
    __shared__ int s_first;
    __shared__ double s_sum[4];
    const int part = blockIdx.x % P.parts, row = blockIdx.x / P.parts, n_target = P.n_drafts + P.n_seqs, lane = threadIdx.x & 63;
    const bool is_t = row < n_target;
    // target rows of sequence b end at cu[b + 1] + b + 1, draft rows at cu[b + 1]
    int seq = 0;
    for (int base = 0; base < P.n_seqs; base += 64) {
        const int i = base + lane;
        const int n = __popcll(__ballot(i < P.n_seqs && (is_t ? P.cu[i + 1] + i + 1 <= row : P.cu[i + 1] <= row - n_target)));
        seq += n;
        if (n < 64) break;
    }
    if (seq >= P.n_seqs) return;                             // behind the last sequence
    const float t = P.temps ? P.temps[seq] : P.temp;
    const T* src = is_t ? (const T*)P.target + (int64_t)row * P.ld_t : (const T*)P.draft + (int64_t)(row - n_target) * P.ld_d;
    const int lo = part * VD_PART, hi = lo + VD_PART < P.vocab ? lo + VD_PART : P.vocab;
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i) load8(src, lo + i * (VD_PART / 2) + 8 * threadIdx.x, hi, x[i]);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, x[i][j]);
    const float top = block_max_f32<4>(m, s_max);
    const double base = top == -INFINITY ? 0.0 : (double)top;    // nothing left in this part: the terms are 0, not NaN
    double sum = 0.0;
    int first = 0x7fffffff;
    if (t > 0.f) {
        const double inv = 1.0 / (double)t;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += exp64(((double)x[i][j] - base) * inv);
    } else {                                                 // the first maximum; a NaN anywhere shows in the sum
        if (threadIdx.x == 0) s_first = 0x7fffffff;
        __syncthreads();
#pragma unroll
        for (int i = 1; i >= 0; --i)
#pragma unroll
            for (int j = 7; j >= 0; --j) {
                if (x[i][j] == top) first = lo + i * (VD_PART / 2) + 8 * threadIdx.x + j;
                sum += x[i][j] != x[i][j] ? NAN : 0.0;
            }
        if (first != 0x7fffffff) atomicMin(&s_first, first);    // a minimum: the order does not matter
        __syncthreads();
        first = s_first;
    }
    sum = block_sum_f64(sum, s_sum);
    if (threadIdx.x == 0) P.stats[(size_t)row * P.parts + part] = RowPart{top, first, sum};
}

// a row's maximum and its first index, and the sum of exponentials relative to it, by one wave
__device__ __forceinline__ void row_total(const VerifyDraftsParams& P, int row, double inv, float& top, int& first, double& sum) {
    const RowPart* s = P.stats + (size_t)row * P.parts;
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int p = lane; p < P.parts; p += 64) m = fmaxf(m, s[p].top);
    top = wave_max_f32_dpp(m);
    double z = 0.0;
    int f = 0x7fffffff;
    for (int p = lane; p < P.parts; p += 64) {
        const RowPart r = s[p];
        if (r.top == top) f = f < r.first ? f : r.first;
        z += r.top == -INFINITY ? r.sum : r.sum * exp64(((double)r.top - (double)top) * inv);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const int w = __shfl_xor(f, o, 64); f = f < w ? f : w; }
    first = f;
    sum = wave_sum_f64(z);
}

struct Walk { int n, at, k; double inv; bool greedy; };

// The accept walk of sequence b (all four waves; the accepted count in every thread), and the totals of the rows that the next
// token is drawn from, in `tot` = {top p, sum p, top q, sum q, first maximum}.
template <typename T>
__device__ __forceinline__ Walk walk(const VerifyDraftsParams& P, int b, double (&tot)[5], int* s_reject, double* s_tot) {
    Walk W;
    W.at = P.cu[b];
    W.n = P.cu[b + 1] - W.at;
    if (W.at < 0 || W.n < 0 || W.at + W.n > P.n_drafts) W.n = -1;
    const float t = P.temps ? P.temps[b] : P.temp;
    W.greedy = !(t > 0.f);
    W.inv = W.greedy ? 0.0 : 1.0 / (double)t;
    W.k = 0;
    if (W.n < 0) return W;
    const int wave = threadIdx.x >> 6, n_target = P.n_drafts + P.n_seqs;
    if (threadIdx.x == 0) *s_reject = W.n;
    __syncthreads();
    for (int i = wave; i < W.n; i += 4) {
        const int64_t tok = P.tokens[W.at + i];
        const int row = W.at + b + i;
        bool ok = false;
        float top; int first; double z;
        row_total(P, row, W.inv, top, first, z);
        if (tok >= 0 && tok < P.vocab) {
            if (W.greedy) {
                ok = top > -INFINITY && z == 0.0 && first == tok;
            } else {
                const double p = exp64(((double)(float)((const T*)P.target)[(int64_t)row * P.ld_t + tok] - (double)top) * W.inv) / z;
                row_total(P, n_target + W.at + i, W.inv, top, first, z);
                const double q = exp64(((double)(float)((const T*)P.draft)[(int64_t)(W.at + i) * P.ld_d + tok] - (double)top) * W.inv) / z;
                ok = (double)P.u_accept[W.at + i] * q < p;
            }
        }
        if (!ok && (threadIdx.x & 63) == 0) atomicMin(s_reject, i);     // a minimum: the order does not matter
    }
    __syncthreads();
    W.k = *s_reject;
    if (wave == 0) {
        float top; int first; double z;
        row_total(P, W.at + b + W.k, W.inv, top, first, z);
        if (threadIdx.x == 0) { s_tot[0] = top; s_tot[1] = z; s_tot[4] = first; }
    } else if (wave == 1) {
        float top = 0.f; int first; double z = 1.0;
        if (W.k < W.n && !W.greedy) row_total(P, n_target + W.at + W.k, W.inv, top, first, z);
        if ((threadIdx.x & 63) == 0) { s_tot[2] = top; s_tot[3] = z; }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 5; ++i) tot[i] = s_tot[i];
    return W;
}

// p and max(p - q, 0) of 8 consecutive tokens
template <typename T>
__device__ __forceinline__ void residual8(const VerifyDraftsParams& P, int b, const Walk& W, const double (&tot)[5], int at, int hi,
                                          double (&p)[8], double (&r)[8]) {
    float x[8], y[8];
    load8((const T*)P.target + (int64_t)(W.at + b + W.k) * P.ld_t, at, hi, x);
    const bool two = W.k < W.n;
    if (two) load8((const T*)P.draft + (int64_t)(W.at + W.k) * P.ld_d, at, hi, y);
    const double ip = 1.0 / tot[1], iq = 1.0 / tot[3];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = at + j < hi ? exp64(((double)x[j] - tot[0]) * W.inv) * ip : 0.0;
        r[j] = p[j];
        if (two) {
            const double d = p[j] - (at + j < hi ? exp64(((double)y[j] - tot[2]) * W.inv) * iq : 0.0);
            r[j] = d < 0.0 ? 0.0 : d;                        // NaN stays
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(VD_THREADS) verify_drafts_walk_kernel(VerifyDraftsParams P) {
    __shared__ int s_reject;
    __shared__ double s_tot[5], s_sum[4];
    const int part = blockIdx.x % P.parts, b = blockIdx.x / P.parts;
    double tot[5];
    const Walk W = walk<T>(P, b, tot, &s_reject, s_tot);
    if (part == 0 && threadIdx.x == 0) {
        P.accepted[b] = W.k;
        if (W.n < 0) P.next[b] = -1;
        else if (W.greedy) P.next[b] = tot[0] > -INFINITY && tot[1] == 0.0 ? (int64_t)tot[4] : -1;
    }
    if (W.n < 0 || W.greedy) return;
    const int lo = part * VD_PART, hi = lo + VD_PART < P.vocab ? lo + VD_PART : P.vocab;
    double all = 0.0, rest = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        double p[8], r[8];
        residual8<T>(P, b, W, tot, lo + i * (VD_PART / 2) + 8 * threadIdx.x, hi, p, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) { all += p[j]; rest += r[j]; }
    }
    rest = block_sum_f64(rest, s_sum);
    all = block_sum_f64(all, s_sum);
    if (threadIdx.x == 0) {
        double* m = P.mass + ((size_t)b * P.parts + part) * 2;
        m[0] = rest;
        m[1] = all;
    }
}

template <typename T>
__global__ void __launch_bounds__(VD_THREADS) verify_drafts_draw_kernel(VerifyDraftsParams P) {
    __shared__ int s_reject, s_hit, s_last, s_part, s_which;
    __shared__ double s_tot[5], s_scan[VD_THREADS], s_base, s_goal;
    const int b = blockIdx.x;
    double tot[5];
    const Walk W = walk<T>(P, b, tot, &s_reject, s_tot);
    if (W.n < 0 || W.greedy) return;                         // decided already
    if (threadIdx.x == 0) {
        const double* m = P.mass + (size_t)b * P.parts * 2;
        double total[2] = {0.0, 0.0};
        for (int p = 0; p < P.parts; ++p) { total[0] += m[2 * p]; total[1] += m[2 * p + 1]; }
        const int which = total[0] == 0.0 ? 1 : 0;           // p nowhere above q: p itself
        const double goal = (double)P.u_next[b] * total[which];
        int part = -1, last = 0;
        double before = 0.0, base = 0.0, last_base = 0.0;
        for (int p = 0; p < P.parts && part < 0; ++p) {
            const double v = m[2 * p + which];
            if (v > 0.0) { last = p; last_base = before; }
            if (before + v > goal) { part = p; base = before; }
            before += v;
        }
        if (part < 0) { part = last; base = last_base; }
        s_part = total[which] > 0.0 && total[which] < INFINITY ? part : -1;     // NaN: no distribution to draw from
        s_base = base; s_goal = goal; s_which = which;
        s_hit = 0x7fffffff; s_last = -1;
    }
    __syncthreads();
    if (s_part < 0) {
        if (threadIdx.x == 0) P.next[b] = -1;
        return;
    }
    const int lo = s_part * VD_PART + VD_EPT * threadIdx.x, hi = (s_part + 1) * VD_PART < P.vocab ? (s_part + 1) * VD_PART : P.vocab;
    double v[VD_EPT], mine = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        double p[8], r[8];
        residual8<T>(P, b, W, tot, lo + 8 * i, hi, p, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) { v[8 * i + j] = s_which ? p[j] : r[j]; mine += v[8 * i + j]; }
    }
    s_scan[threadIdx.x] = mine;                              // inclusive scan over the threads
    __syncthreads();
#pragma unroll
    for (int o = 1; o < VD_THREADS; o <<= 1) {
        const double add = threadIdx.x >= o ? s_scan[threadIdx.x - o] : 0.0;
        __syncthreads();
        s_scan[threadIdx.x] += add;
        __syncthreads();
    }
    double run = s_base + (threadIdx.x ? s_scan[threadIdx.x - 1] : 0.0);
    int hit = 0x7fffffff, last = -1;
#pragma unroll
    for (int j = 0; j < VD_EPT; ++j) {
        run += v[j];
        if (v[j] > 0.0) {
            last = lo + j;
            if (run > s_goal && hit == 0x7fffffff) hit = lo + j;
        }
    }
    if (hit != 0x7fffffff) atomicMin(&s_hit, hit);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (threadIdx.x == 0) P.next[b] = s_hit != 0x7fffffff ? s_hit : s_last;     // the last one that has mass, where rounding left none
}

extern "C" size_t sq_verify_drafts_workspace_bytes(int n_seqs, int n_drafts, int vocab) {
    if (n_seqs <= 0 || n_drafts < 0 || vocab <= 0) return 0;
    const size_t parts = ((size_t)vocab + VD_PART - 1) / VD_PART;
    return parts * (((size_t)2 * n_drafts + n_seqs) * sizeof(RowPart) + (size_t)n_seqs * 2 * sizeof(double));
}

extern "C" int sq_verify_drafts(const void* target_logits, int64_t ld_target, const void* draft_logits, int64_t ld_draft,
                                const int64_t* d_draft_tokens, const int32_t* d_cu_drafts, int n_seqs, int n_drafts, int vocab,
                                const float* d_u_accept, const float* d_u_next, const float* d_temperature, float temperature,
                                int32_t* d_n_accepted, int64_t* d_next_tokens, int dtype, void* workspace, size_t workspace_bytes,
                                void* stream) {
    if (n_seqs < 0 || n_drafts < 0 || vocab <= 0) return SQ_EINVAL;
    if (dtype != SQ_DTYPE_F16 && dtype != SQ_DTYPE_BF16 && dtype != SQ_DTYPE_F32) return SQ_EUNSUPPORTED;
    if (n_seqs == 0) return SQ_OK;
    if (!target_logits || !d_cu_drafts || !d_u_next || !d_n_accepted || !d_next_tokens || ld_target < vocab) return SQ_EINVAL;
    if (n_drafts && (!draft_logits || !d_draft_tokens || !d_u_accept || ld_draft < vocab)) return SQ_EINVAL;
    if (!d_temperature && !(temperature >= 0.f && temperature < INFINITY)) return SQ_EINVAL;
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < sq_verify_drafts_workspace_bytes(n_seqs, n_drafts, vocab)) return SQ_EINVAL;
    const int parts = (vocab + VD_PART - 1) / VD_PART;
    const int64_t rows = 2 * (int64_t)n_drafts + n_seqs;
    if (rows * parts > 0x7fffffff) return SQ_EUNSUPPORTED;
    RowPart* stats = (RowPart*)workspace;
    VerifyDraftsParams P = {target_logits, draft_logits, ld_target, ld_draft, d_draft_tokens, d_cu_drafts, d_u_accept, d_u_next, d_temperature,
                            temperature, d_n_accepted, d_next_tokens, n_seqs, n_drafts, vocab, parts, stats, (double*)(stats + rows * parts)};
    hipStream_t st = (hipStream_t)stream;
#define SQ_V(TT) do { \
        hipLaunchKernelGGL((verify_drafts_stats_kernel<TT>), dim3((unsigned)(rows * parts)), dim3(VD_THREADS), 0, st, P); \
        hipLaunchKernelGGL((verify_drafts_walk_kernel<TT>), dim3((unsigned)(n_seqs * parts)), dim3(VD_THREADS), 0, st, P); \
        hipLaunchKernelGGL((verify_drafts_draw_kernel<TT>), dim3((unsigned)n_seqs), dim3(VD_THREADS), 0, st, P); \
    } while (0)
    if (dtype == SQ_DTYPE_F16) SQ_V(half_t);
    else if (dtype == SQ_DTYPE_BF16) SQ_V(bf16_t);
    else SQ_V(float);
#undef SQ_V
    return sq_check_launch();
}
