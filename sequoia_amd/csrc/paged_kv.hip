// Rows into and out of a paged KV cache: RoPE + write of a ragged batch's new tokens (16-bit rows, or e4m3 rows with an exponent
// byte each), and the read of stored rows into the static slab layout.  Both move bytes and nothing else: one pass, 16-byte
// accesses, everything that does not depend on a load issued before it.
#include "paged.h"

#define PKV_THREADS 256

struct PagedWriteParams {
    const void* qkv; int64_t qkv_stride;
    void* q_out;
    void *k, *v;
    uint8_t *ks, *vs;
    const void *cos, *sin;
    int max_pos;
    const int64_t* pos;
    PageMap map;
    const int32_t *seq_lens, *cu_rows;
    int n_seqs, n_rows, n_heads, h_kv;
};

// One workgroup: one token, PKV_THREADS / (D / 16) of its H + 2 H_kv head rows.  A lane holds elements [8c, 8c + 8) of both halves
// of its row, so the rotation (o1 = x1 cos - x2 sin, o2 = x2 cos + x1 sin) is lane-local and a row's largest magnitude takes
// log2(D / 16) lane exchanges.  The products of two 16-bit values are exact in fp32; the one rounding of the sum is followed by
// the one to the stored type.
// Bound by bytes, read once and written once, and by latency below about a hundred rows: 6730 rows of 64 + 2 * 8 heads of 128, fp16,
// 51 us (5.5 TB/s, a large copy here reaches 5.1; 42 where the call before read the same rows, which the last-level cache then holds in
// part); 32 rows into e4m3 pages 3.6 us, a call 4.4.  The stores go past the caches: cached ones took 55.6 us, and the attention that
// reads the rows next, mostly on another XCD, takes the same time.
template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(PKV_THREADS) rope_kv_write_paged_kernel(PagedWriteParams P) {
    typedef typename vec_of<T>::v8 v8;
    constexpr int LPR = D / 16, RPB = PKV_THREADS / LPR;
    const int t = blockIdx.x, unit = blockIdx.y * RPB + threadIdx.x / LPR, c = threadIdx.x % LPR;
    const int units = P.n_heads + 2 * P.h_kv;
    const bool live = unit < units;                       // the last workgroup of a token: lanes past its rows stay for the exchanges
    const T* row = (const T*)P.qkv + (size_t)t * P.qkv_stride + (size_t)(live ? unit : 0) * D + 8 * c;
    const v8 a8 = *(const v8*)row, b8 = *(const v8*)(row + D / 2);
    int64_t pos = P.pos[t];
    pos = pos < 0 ? 0 : (pos >= P.max_pos ? P.max_pos - 1 : pos);         // in bounds whatever the caller's ids hold
    const int seq = seq_of_row(P.cu_rows, P.n_seqs, t);
    if (seq >= P.n_seqs || P.cu_rows[seq] > t) return;    // a row of no sequence (uniform): left alone
    float x1[8], x2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { x1[j] = (float)a8[j]; x2[j] = (float)b8[j]; }
    if (unit < P.n_heads + P.h_kv) {
        const T *cr = (const T*)P.cos + (size_t)pos * D + 8 * c, *sr = (const T*)P.sin + (size_t)pos * D + 8 * c;
        const v8 c1 = *(const v8*)cr, c2 = *(const v8*)(cr + D / 2), s1 = *(const v8*)sr, s2 = *(const v8*)(sr + D / 2);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float u = x1[j], w = x2[j];
            x1[j] = u * (float)c1[j] - w * (float)s1[j];
            x2[j] = w * (float)c2[j] + u * (float)s2[j];
        }
    }
    v8 o1, o2;
    if (unit < P.n_heads) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { o1[j] = (T)x1[j]; o2[j] = (T)x2[j]; }
        T* dst = (T*)P.q_out + ((size_t)unit * P.n_rows + t) * D + 8 * c;
        __builtin_nontemporal_store(o1, (v8*)dst);
        __builtin_nontemporal_store(o2, (v8*)(dst + D / 2));
    }
    const bool is_v = unit >= P.n_heads + P.h_kv;
    const int kvh = unit - P.n_heads - (is_v ? P.h_kv : 0);
    const int slot = P.seq_lens[seq] + (t - P.cu_rows[seq]);
    const int page = slot < 0 ? -1 : page_of(P.map, seq, slot >> P.map.shift);
    const bool store = live && unit >= P.n_heads && page >= 0;
    const size_t r = (((size_t)(page < 0 ? 0 : page) * P.h_kv + (kvh < 0 ? 0 : kvh)) << P.map.shift) + (slot & ((1 << P.map.shift) - 1));
    if constexpr (!Q8) {
        if (!store) return;
#pragma unroll
        for (int j = 0; j < 8; ++j) { o1[j] = (T)x1[j]; o2[j] = (T)x2[j]; }
        T* dst = (T*)(is_v ? P.v : P.k) + r * D + 8 * c;
        __builtin_nontemporal_store(o1, (v8*)dst);
        __builtin_nontemporal_store(o2, (v8*)(dst + D / 2));
    } else {
        // Magnitudes stop at the largest value of T that has four significant bits: one more step would read back as infinity.
        // An element that is not finite is stored as NaN and has no part in the scale.
        const float top = __is_same(T, half_t) ? 61440.0f : 0x1.ep127f;
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float m1 = __builtin_fabsf(x1[j]), m2 = __builtin_fabsf(x2[j]);
            big = fmaxf(big, fmaxf(m1 < INFINITY ? m1 : 0.f, m2 < INFINITY ? m2 : 0.f));
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
        if (!store) return;
        // smallest x with big * 2^(127 - x) <= 448 = 1.75 * 2^8, from the bits of big
        const uint32_t bits = __builtin_bit_cast(uint32_t, fminf(big, top));
        int x = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
        x = x < 1 ? 1 : x;
        const float inv = e4m3_scale(254 - x);
        u32x2 w1, w2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float y1[4], y2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = x1[4 * h + j], w = x2[4 * h + j];
                y1[j] = __builtin_fabsf(u) < INFINITY ? fminf(fmaxf(u, -top), top) * inv : NAN;
                y2[j] = __builtin_fabsf(w) < INFINITY ? fminf(fmaxf(w, -top), top) * inv : NAN;
            }
            w1[h] = __builtin_amdgcn_cvt_pk_fp8_f32(y1[2], y1[3], __builtin_amdgcn_cvt_pk_fp8_f32(y1[0], y1[1], 0, false), true);
            w2[h] = __builtin_amdgcn_cvt_pk_fp8_f32(y2[2], y2[3], __builtin_amdgcn_cvt_pk_fp8_f32(y2[0], y2[1], 0, false), true);
        }
        uint8_t* dst = (uint8_t*)(is_v ? P.v : P.k) + r * D + 8 * c;
        __builtin_nontemporal_store(w1, (u32x2*)dst);
        __builtin_nontemporal_store(w2, (u32x2*)(dst + D / 2));
        if (c == 0) (is_v ? P.vs : P.ks)[r] = (uint8_t)x;
    }
}

extern "C" int sq_rope_kv_write_paged(const void* qkv, int64_t qkv_stride, void* q_out, void* k_pages, void* v_pages, void* k_scales,
                                      void* v_scales, const void* cos_tab, const void* sin_tab, int max_pos,
                                      const int64_t* d_position_ids, const int32_t* d_page_table, int table_width, int n_pages,
                                      int page_size, const int32_t* d_seq_lens, const int32_t* d_cu_rows, int n_seqs, int n_rows,
                                      int n_heads, int h_kv, int d, int dtype, void* stream) {
    if (n_seqs < 0 || n_rows < 0 || n_heads <= 0 || h_kv <= 0 || n_heads % h_kv || max_pos <= 0 || table_width < 0 || n_pages <= 0)
        return SQ_EINVAL;
    if (!k_scales != !v_scales) return SQ_EINVAL;
    const int shift = page_shift(page_size);
    if ((d != 64 && d != 128) || shift < 0 || (dtype != SQ_DTYPE_F16 && dtype != SQ_DTYPE_BF16)) return SQ_EUNSUPPORTED;
    if (n_rows == 0 || n_seqs == 0) return SQ_OK;
    if (!qkv || !q_out || !k_pages || !v_pages || !cos_tab || !sin_tab || !d_position_ids || !d_page_table || !d_seq_lens || !d_cu_rows)
        return SQ_EINVAL;
    if (qkv_stride < (int64_t)(n_heads + 2 * h_kv) * d || (qkv_stride & 7)) return SQ_EINVAL;
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15) return SQ_EINVAL;
    PagedWriteParams P = {qkv, qkv_stride, q_out, k_pages, v_pages, (uint8_t*)k_scales, (uint8_t*)v_scales, cos_tab, sin_tab, max_pos,
                          d_position_ids, {d_page_table, table_width, n_pages, shift}, d_seq_lens, d_cu_rows, n_seqs, n_rows, n_heads, h_kv};
    const int rpb = PKV_THREADS / (d / 16);
    const dim3 grid(n_rows, (n_heads + 2 * h_kv + rpb - 1) / rpb);
    if (grid.x > PAGED_MAX_GRID || grid.y > 65535) return SQ_EUNSUPPORTED;
    hipStream_t st = (hipStream_t)stream;
#define SQ_W(TT, DD, QQ) hipLaunchKernelGGL((rope_kv_write_paged_kernel<TT, DD, QQ>), grid, dim3(PKV_THREADS), 0, st, P)
#define SQ_WD(TT, DD) do { if (k_scales) SQ_W(TT, DD, true); else SQ_W(TT, DD, false); } while (0)
    if (dtype == SQ_DTYPE_F16) { if (d == 128) SQ_WD(half_t, 128); else SQ_WD(half_t, 64); }
    else                       { if (d == 128) SQ_WD(bf16_t, 128); else SQ_WD(bf16_t, 64); }
#undef SQ_WD
#undef SQ_W
    return sq_check_launch();
}

struct PagedReadParams {
    const void *k, *v;
    const uint8_t *ks, *vs;
    void *k_out, *v_out;
    int64_t seq_stride, head_stride;    // of the outputs, in elements; a row is D contiguous elements
    int out_rows;
    PageMap map;
    const int32_t *starts, *counts;
    int n_blocks, h_kv;                 // workgroups over a sequence's rows
};

// One workgroup: PKV_READ_ROWS rows of one (sequence, KV head), K and V.  A lane moves eight elements of a row at a time, so that
// loads and stores both cover whole lines, every pass's loads issued before the first store; the rows go past the caches, other
// layers' come before anybody reads them.  Bound by bytes: eight sequences of 700-9000 e4m3 rows of 8 heads of 128 to bf16, 33.6 us
// (6.2 TB/s; cached stores 45; sixteen codes a lane, whose two stores leave every other 16 bytes to each other, 48; 64 rows a workgroup
// 49, loads past the caches too 41).  One sequence of 230 rows: 2.7 us, a call 4.3.
template <bool Q8> struct stored8 { typedef u32x4 type; };
template <> struct stored8<true> { typedef u32x2 type; };
#define PKV_READ_ROWS 32
template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(PKV_THREADS) kv_read_paged_kernel(PagedReadParams P) {
    typedef typename vec_of<T>::v8 v8;
    typedef typename stored8<Q8>::type piece;
    constexpr int LPR = D / 8;                                        // lanes a row
    constexpr int RPP = PKV_THREADS / LPR;                            // rows a pass
    constexpr int PASSES = PKV_READ_ROWS > RPP ? PKV_READ_ROWS / RPP : 1;
    const int blk = blockIdx.x % P.n_blocks, bh = blockIdx.x / P.n_blocks, h = bh % P.h_kv, b = bh / P.h_kv;
    int n = P.counts[b];
    n = n < P.out_rows ? n : P.out_rows;
    const int first = blk * (PASSES * RPP) + threadIdx.x / LPR, c = threadIdx.x % LPR, start = P.starts[b];
    piece kr[PASSES], vr[PASSES];
    uint32_t ks[PASSES], vs[PASSES];
    bool ok[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int j = first + i * RPP, slot = start + j;
        const int page = j < n && slot >= 0 ? page_of(P.map, b, slot >> P.map.shift) : -1;
        ok[i] = page >= 0;
        if (ok[i]) {
            const size_t r = (((size_t)page * P.h_kv + h) << P.map.shift) + (slot & ((1 << P.map.shift) - 1));
            const size_t at = (r * D + 8 * c) * (Q8 ? 1 : 2);
            kr[i] = *(const piece*)((const uint8_t*)P.k + at);
            vr[i] = *(const piece*)((const uint8_t*)P.v + at);
            if constexpr (Q8) { ks[i] = P.ks[r]; vs[i] = P.vs[r]; }
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        if (!ok[i]) continue;
        const size_t at = (size_t)b * P.seq_stride + (size_t)h * P.head_stride + (size_t)(first + i * RPP) * D + 8 * c;
        T *kd = (T*)P.k_out + at, *vd = (T*)P.v_out + at;
        if constexpr (Q8) {
            v8 lo, hi;
            e4m3_expand<T>(u32x4{kr[i][0], kr[i][1], 0, 0}, e4m3_scale(ks[i]), lo, hi);
            __builtin_nontemporal_store(lo, (v8*)kd);
            e4m3_expand<T>(u32x4{vr[i][0], vr[i][1], 0, 0}, e4m3_scale(vs[i]), lo, hi);
            __builtin_nontemporal_store(lo, (v8*)vd);
        } else {
            __builtin_nontemporal_store(kr[i], (piece*)kd);
            __builtin_nontemporal_store(vr[i], (piece*)vd);
        }
    }
}

extern "C" int sq_kv_read_paged(const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, void* k_out,
                                void* v_out, int64_t out_seq_stride, int64_t out_head_stride, int out_rows,
                                const int32_t* d_page_table, int table_width, int n_pages, int page_size, const int32_t* d_starts,
                                const int32_t* d_counts, int n_seqs, int max_count, int h_kv, int d, int dtype, void* stream) {
    if (n_seqs < 0 || max_count < 0 || out_rows < 0 || h_kv <= 0 || table_width < 0 || n_pages <= 0) return SQ_EINVAL;
    if (!k_scales != !v_scales) return SQ_EINVAL;
    const int shift = page_shift(page_size);
    if ((d != 64 && d != 128) || shift < 0 || (dtype != SQ_DTYPE_F16 && dtype != SQ_DTYPE_BF16)) return SQ_EUNSUPPORTED;
    if (max_count > out_rows) max_count = out_rows;
    if (n_seqs == 0 || max_count == 0) return SQ_OK;
    if (!k_pages || !v_pages || !k_out || !v_out || !d_page_table || !d_starts || !d_counts) return SQ_EINVAL;
    if (((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return SQ_EINVAL;
    if (((out_seq_stride | out_head_stride) & 7) || out_head_stride < (int64_t)out_rows * d) return SQ_EINVAL;
    const int rpp = PKV_THREADS / (d / 8), per = rpp > PKV_READ_ROWS ? rpp : PKV_READ_ROWS;
    const int n_blocks = (max_count + per - 1) / per;
    const int64_t grid = (int64_t)n_blocks * h_kv * n_seqs;
    if (grid > PAGED_MAX_GRID) return SQ_EUNSUPPORTED;
    PagedReadParams P = {k_pages, v_pages, (const uint8_t*)k_scales, (const uint8_t*)v_scales, k_out, v_out, out_seq_stride,
                         out_head_stride, max_count, {d_page_table, table_width, n_pages, shift}, d_starts, d_counts, n_blocks, h_kv};
    hipStream_t st = (hipStream_t)stream;
#define SQ_R(TT, DD, QQ) hipLaunchKernelGGL((kv_read_paged_kernel<TT, DD, QQ>), dim3((unsigned)grid), dim3(PKV_THREADS), 0, st, P)
#define SQ_RD(TT, DD) do { if (k_scales) SQ_R(TT, DD, true); else SQ_R(TT, DD, false); } while (0)
    if (dtype == SQ_DTYPE_F16) { if (d == 128) SQ_RD(half_t, 128); else SQ_RD(half_t, 64); }
    else                       { if (d == 128) SQ_RD(bf16_t, 128); else SQ_RD(bf16_t, 64); }
#undef SQ_RD
#undef SQ_R
    return sq_check_launch();
}
