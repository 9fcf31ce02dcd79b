// Attention of a ragged batch's new tokens over a paged KV cache (their own rows already written): for sequence b with `past`
// stored rows and n new ones, row i attends keys [0, past + i],
//     o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale * q . k_j,
// in one pass over the keys with a running maximum and sum in fp32; weights are rounded to the element type once, for the
// second matrix product.  The query heads that share a KV head are packed into the same rows of a tile (row r = token r / group,
// head r % group), so that every stored row is read once for all of them.
#include "paged.h"
#include "attn_map.h"

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __fp16 fp16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));

// Values loaded before a loop are waited for before it: left to the loop, the wait for them is repeated in every trip, and there it
// is a wait for the trip's own prefetch.
template <typename V> __device__ __forceinline__ void arrived(V& v) { asm volatile("" : "+v"(v)); }

struct PagedAttnParams {
    const void* q; int64_t q_head_stride, q_row_stride;
    const void *k, *v;
    const uint8_t *ks, *vs;
    void* out; int64_t out_stride;
    PageMap map;
    const int32_t *seq_lens, *cu_rows;
    int n_seqs, n_rows, n_heads, h_kv, group;
    float scale_log2e;
    int max_len;                           // no sequence's keys go further (host's bound: the parts cover it)
    int n_tiles, n_splits, split_len;      // row tiles a (sequence, KV head), parts of the key axis, keys a part
    float* part_o;                         // [n_splits][n_rows * n_heads][D]: unnormalised
    float* part_ml;                        // [n_splits][n_rows * n_heads][2]: maximum (log2 units), sum
};

template <typename T> __device__ __forceinline__ floatx4 mfma16(typename vec_of<T>::v8 a, typename vec_of<T>::v8 b, floatx4 c) {
    if constexpr (__is_same(T, half_t)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <typename T> __device__ __forceinline__ floatx16 mfma32(typename vec_of<T>::v8 a, typename vec_of<T>::v8 b, floatx16 c) {
    if constexpr (__is_same(T, half_t)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// column (lane & 15) of the 4 x 16 block of 16-bit values whose row (lane & 15) >> 2, columns 4 (lane & 3).. this lane addresses
__device__ __forceinline__ u32x2 read_transposed(const void* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)p));
}

// A weight of 0 must not meet an infinity or a NaN in a row of V that some query does not see.  Where a chunk of keys holds such
// rows, what is not finite is staged as 0 and its rows are noted; add_hidden puts it back for the queries that do see it.
// Returns whether anything of v was not finite (an exponent of all ones: adding one to it carries into the sign's place).
template <typename T> __device__ __forceinline__ bool take_nonfinite(typename vec_of<T>::v8& v) {
    constexpr uint32_t E = __is_same(T, half_t) ? 0x7c007c00u : 0x7f807f80u, ONE = __is_same(T, half_t) ? 0x04000400u : 0x00800080u;
    u32x4 w = __builtin_bit_cast(u32x4, v);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bad = ((w[i] & E) + ONE) & 0x80008000u;
        any |= bad;
        w[i] &= ~(bad | (bad - (bad >> 15)));
    }
    v = __builtin_bit_cast(typename vec_of<T>::v8, w);
    return any != 0;
}
// the four elements of a stored row of V from column d on, those that are finite as 0
template <typename T, int D, bool Q8> __device__ __forceinline__ void hidden4(const PagedAttnParams& P, size_t row, int d, float (&x)[4]) {
    if constexpr (Q8) {
        const uint32_t w = *(const uint32_t*)((const uint8_t*)P.v + row * D + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = ((w >> (8 * j)) & 0x7fu) == 0x7fu ? NAN : 0.f;
    } else {
        const typename vec_of<T>::v4 w = *(const typename vec_of<T>::v4*)((const T*)P.v + row * D + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __builtin_fabsf((float)w[j]) < INFINITY ? 0.f : (float)w[j];
    }
}

// 16 bytes a lane from base + from (base uniform) to LDS byte to + 16 * lane (uniform).  By hand, because the compiler takes any LDS
// read for one of what such a load writes, and waits for all of them in front of it: who reads the bytes calls loads_done() first.
__device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(from), "s"(base), "s"(to) : "memory");      // (m0 is nobody else's here)
}
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// what a workgroup works on
struct AttnItem {
    int seq, kvh, past, rows, first, row0, end, split, n_parts;   // packed rows of the (sequence, KV head), cu_rows[seq], first row, key end
};
__device__ __forceinline__ int attn_tile_end(const PagedAttnParams& P, int past, int rows, int tile, int tile_rows) {
    int last = (tile + 1) * tile_rows;
    last = last < rows ? last : rows;
    const int end = past + (last - 1) / P.group + 1;
    return end < P.max_len ? (end > 0 ? end : 0) : P.max_len;
}
// (sequence, KV head) fastest: a multiple of 8 of them keeps all tiles of one in one XCD's L2; the longest tiles start first
__device__ __forceinline__ bool attn_item(const PagedAttnParams& P, int tile_rows, AttnItem& I) {
    const int units = P.n_seqs * P.h_kv, u = blockIdx.x % units, w = blockIdx.x / units;
    I.seq = u / P.h_kv; I.kvh = u - I.seq * P.h_kv;
    const int tile = P.n_tiles - 1 - w / P.n_splits;
    I.split = w % P.n_splits;
    I.first = __builtin_amdgcn_readfirstlane(P.cu_rows[I.seq]);        // scalar registers: what branches on these is uniform
    const int n = __builtin_amdgcn_readfirstlane(P.cu_rows[I.seq + 1]) - I.first;
    I.past = __builtin_amdgcn_readfirstlane(P.seq_lens[I.seq]);
    if (I.first < 0 || I.first + n > P.n_rows) return false;
    I.rows = n * P.group;
    I.row0 = tile * tile_rows;
    if (I.row0 >= I.rows) return false;
    I.end = attn_tile_end(P, I.past, I.rows, tile, tile_rows);
    I.n_parts = (I.end + P.split_len - 1) / P.split_len;
    return I.split < I.n_parts || (I.split == 0 && I.n_parts == 0);
}

__device__ __forceinline__ size_t stored_row(const PagedAttnParams& P, int page, int kvh, int key) {
    return (((size_t)page * P.h_kv + kvh) << P.map.shift) + (key & ((1 << P.map.shift) - 1));
}

// Few rows (a decoding step, a drafted chunk): bound by the bytes of K and V.  Four waves walk the 32-key chunks of the
// workgroup's part in turn, each with its own running softmax, and join through LDS.  A chunk is fetched as whole rows (16 bytes
// a lane, next chunk in flight while this one is computed), staged in the wave's own LDS and read back as
//   S^T = K Q^T    A = K rows, B = Q: a lane holds 8 scores of one query row, in the order the second product wants them
//   O^T += V^T P^T A = V^T (transposing LDS reads), B = P^T straight from the registers S^T left behind.
#define PAD_NW 4
#define PAD_BK 32
template <typename T, int D, bool Q8, int MT>
__global__ void __launch_bounds__(PAD_NW * 64, 2) paged_attention_rows_kernel(PagedAttnParams P) {
    typedef typename vec_of<T>::v8 v8;
    typedef typename vec_of<T>::v4 v4;
    constexpr int EPL = Q8 ? 16 : 8, LPR = D / EPL, RPP = 64 / LPR, PASSES = PAD_BK / RPP;   // elements a lane, lanes a row, rows a pass
    constexpr int DSTEPS = D / 32, NT = D / 16, ROWS = 16 * MT;
    constexpr int KSTR = D + 8, VSTR = D + 16;      // 16-byte reads of 16 rows, 8-byte transposing reads of 8 rows: all banks once
    constexpr int WAVE_BYTES = PAD_BK * (KSTR + VSTR) * 2, OSTR = D + 4;
    constexpr int LDS_BYTES = PAD_NW * (WAVE_BYTES > ROWS * OSTR * 4 ? WAVE_BYTES : ROWS * OSTR * 4);
    __shared__ __attribute__((aligned(16))) unsigned char lds[LDS_BYTES];
    __shared__ float lds_ml[PAD_NW][ROWS][2];
    AttnItem I;
    if (!attn_item(P, ROWS, I)) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qc = lane & 15, g = lane >> 4;
    const int k0 = I.split * P.split_len, k1 = I.end < k0 + P.split_len ? I.end : k0 + P.split_len;
    T* my_k = (T*)(lds + wave * WAVE_BYTES);
    T* my_v = my_k + PAD_BK * KSTR;

    v8 qf[MT][DSTEPS];
    int lim[MT];                                    // last key this lane's query row sees
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        int r = I.row0 + 16 * mt + qc;
        r = r < I.rows ? r : I.rows - 1;
        const int token = r / P.group, head = I.kvh * P.group + r - token * P.group;
        lim[mt] = I.past + token;
        const T* qr = (const T*)P.q + head * P.q_head_stride + (size_t)(I.first + token) * P.q_row_stride + 8 * g;
#pragma unroll
        for (int s = 0; s < DSTEPS; ++s) qf[mt][s] = *(const v8*)(qr + 32 * s);
    }
    const int lim0 = I.past + I.row0 / P.group;     // keys up to here are seen by every row of the tile

    float m_run[MT], l_run[MT];
    floatx4 o_acc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m_run[mt] = -INFINITY; l_run[mt] = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) o_acc[mt][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    u32x4 kr[PASSES], vr[PASSES];
    uint32_t ksr[PASSES], vsr[PASSES];
    const int lrow = lane / LPR, lcol = lane % LPR;
    // entries of the pages that hold the two 16-row halves of a chunk
    auto pages = [&](int key0, int& a, int& b) {
        a = page_entry(P.map, I.seq, key0 >> P.map.shift);
        b = page_entry(P.map, I.seq, (key0 + 16) >> P.map.shift);
    };
    auto load = [&](int key0, int ea, int eb) {
        const size_t ra = stored_row(P, check_page(P.map, ea), I.kvh, key0), rb = stored_row(P, check_page(P.map, eb), I.kvh, key0 + 16);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const size_t r = i * RPP < 16 ? ra + i * RPP : rb + (i * RPP - 16);         // scalar
            const uint32_t at = lane * 16;                                              // rows lie one behind the other
            kr[i] = *(const u32x4*)((const uint8_t*)P.k + r * (D * (Q8 ? 1 : 2)) + at);
            vr[i] = *(const u32x4*)((const uint8_t*)P.v + r * (D * (Q8 ? 1 : 2)) + at);
            if constexpr (Q8) { ksr[i] = (P.ks + r)[lrow]; vsr[i] = (P.vs + r)[lrow]; }
        }
    };
    constexpr int STEP = PAD_NW * PAD_BK;
    int key0 = k0 + wave * PAD_BK, ea = 0, eb = 0;
    if (key0 < k1) {
        int fa, fb;
        pages(key0, fa, fb);
        pages(key0 + STEP, ea, eb);
        load(key0, fa, fb);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int s = 0; s < DSTEPS; ++s) arrived(qf[mt][s]);
    for (; key0 < k1; key0 += STEP) {
        const bool tail = key0 + PAD_BK > k1;       // rows behind the end hold anything: their weights are 0, and so are they
        const bool masked = tail || key0 + PAD_BK - 1 > lim0;
        uint32_t hidden = 0;                        // rows of the chunk with values that were taken out
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int rr = i * RPP + lrow;
            bool bad = false;
            if constexpr (Q8) {
                v8 lo, hi;
                e4m3_expand<T>(kr[i], e4m3_scale(ksr[i]), lo, hi);
                *(v8*)(my_k + rr * KSTR + 16 * lcol) = lo;
                *(v8*)(my_k + rr * KSTR + 16 * lcol + 8) = hi;
                if (tail && key0 + rr >= k1) { vr[i] = u32x4{0, 0, 0, 0}; vsr[i] = 127; }
                e4m3_expand<T>(vr[i], e4m3_scale(vsr[i]), lo, hi);
                if (masked) bad = take_nonfinite<T>(lo) | take_nonfinite<T>(hi);
                *(v8*)(my_v + rr * VSTR + 16 * lcol) = lo;
                *(v8*)(my_v + rr * VSTR + 16 * lcol + 8) = hi;
            } else {
                *(u32x4*)(my_k + rr * KSTR + 8 * lcol) = kr[i];
                if (tail && key0 + rr >= k1) vr[i] = u32x4{0, 0, 0, 0};
                v8 w = __builtin_bit_cast(v8, vr[i]);
                if (masked) bad = take_nonfinite<T>(w);
                *(v8*)(my_v + rr * VSTR + 8 * lcol) = w;
            }
            if (masked) {
                const uint64_t lanes = __ballot(bad);
                if (lanes)
                    for (int j = 0; j < RPP; ++j) hidden |= (uint32_t)(((lanes >> (j * LPR)) & ((1ull << LPR) - 1)) != 0) << (i * RPP + j);
            }
        }
        if (key0 + STEP < k1) {                     // the entries of the chunk after the next come first: loads end in order
            const int fa = ea, fb = eb;
            pages(key0 + 2 * STEP, ea, eb);
            load(key0 + STEP, fa, fb);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        floatx4 s_acc[MT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            v8 kf[DSTEPS];
#pragma unroll
            for (int s = 0; s < DSTEPS; ++s) kf[s] = *(const v8*)(my_k + (16 * t + qc) * KSTR + 32 * s + 8 * g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < DSTEPS; ++s) acc = mfma16<T>(kf[s], qf[mt][s], acc);
                s_acc[mt][t] = acc;
            }
        }
        v8 pf[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float sv[8], cmax = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) sv[j] = s_acc[mt][j >> 2][j & 3] * P.scale_log2e;
            if (masked) {
                int seen = (lim[mt] < k1 ? lim[mt] : k1 - 1) - key0 - 4 * g;       // opaque: not eight differences kept over the loop
                asm("" : "+v"(seen));
#pragma unroll
                for (int j = 0; j < 8; ++j) sv[j] = 16 * (j >> 2) + (j & 3) <= seen ? sv[j] : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) cmax = fmaxf(cmax, sv[j]);
            cmax = group4_max(cmax);
            const float m_new = fmaxf(m_run[mt], cmax);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;       // nothing seen so far
            if (__any(m_new > m_run[mt])) {
                const float alpha = __builtin_amdgcn_exp2f(m_run[mt] - m_use);
                l_run[mt] *= alpha;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) o_acc[mt][nt] *= alpha;
                m_run[mt] = m_new;
            }
            float psum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(sv[j] - m_use);
                psum += p;
                pf[mt][j] = (T)p;
            }
            l_run[mt] += psum;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const T* a0 = my_v + (4 * g + (qc >> 2)) * VSTR + 16 * nt + 4 * (qc & 3);
            const u32x2 lo = read_transposed(a0), hi = read_transposed(a0 + 16 * VSTR);
            const v8 vf = __builtin_bit_cast(v8, u32x4{lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) o_acc[mt][nt] = mfma16<T>(vf, pf[mt], o_acc[mt][nt]);
        }
        while (hidden) {                            // wave-uniform, and hardly ever entered
            const int key = key0 + __builtin_ctz(hidden);
            hidden &= hidden - 1;
            const size_t row = stored_row(P, check_page(P.map, page_entry(P.map, I.seq, key >> P.map.shift)), I.kvh, key);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x[4];
                hidden4<T, D, Q8>(P, row, 16 * nt + 4 * g, x);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o_acc[mt][nt][j] += key <= lim[mt] ? x[j] : 0.f;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }

    // ---- join the waves -------------------------------------------------------------------------
    __syncthreads();                                // everyone is done with the staging area
    float* lds_o = (float*)lds;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float l = group4_sum(l_run[mt]);
        if (g == 0) { lds_ml[wave][16 * mt + qc][0] = m_run[mt]; lds_ml[wave][16 * mt + qc][1] = l; }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *(floatx4*)(lds_o + (wave * ROWS + 16 * mt + qc) * OSTR + 16 * nt + 4 * g) = o_acc[mt][nt];
    }
    __syncthreads();
    for (int e = tid; e < ROWS * (D / 4); e += PAD_NW * 64) {
        const int row = e / (D / 4), col = 4 * (e % (D / 4)), r = I.row0 + row;
        if (r >= I.rows) break;                     // rows ascend with e
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < PAD_NW; ++w) m = fmaxf(m, lds_ml[w][row][0]);
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PAD_NW; ++w) {
            const float mw = lds_ml[w][row][0], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
            l += lds_ml[w][row][1] * f;
            o += *(const floatx4*)(lds_o + (w * ROWS + row) * OSTR + col) * f;
        }
        const int token = r / P.group, head = I.kvh * P.group + r - token * P.group;
        if (I.n_parts <= 1) {
            const float inv = l != 0.f ? 1.0f / l : 0.f;            // a row that sees nothing: zeros
            v4 res;
#pragma unroll
            for (int j = 0; j < 4; ++j) res[j] = (T)(o[j] * inv);
            *(v4*)((T*)P.out + (size_t)(I.first + token) * P.out_stride + (size_t)head * D + col) = res;
        } else {
            const size_t pr = ((size_t)I.split * P.n_rows + I.first + token) * P.n_heads + head;
            *(floatx4*)(P.part_o + pr * D + col) = o;
            if (col == 0) { P.part_ml[pr * 2] = m; P.part_ml[pr * 2 + 1] = l; }
        }
    }
}

// Many rows (a prompt's chunk, a wide tree of shared heads): bound by the matrix products and the exponentials between them.  A
// workgroup's four waves hold 32 rows each and share 64-key tiles of K and V in LDS (two buffers: the next tile's rows travel
// global -> registers while this one is computed, registers -> LDS behind it; one barrier a tile).  With 32 x 32 products,
//   S^T = K Q^T    leaves a lane with 32 scores of ONE row: its maximum and sum are lane-local but for one exchange between the
//                  two half-waves, and the weights are the second product's B operand where they stand
//   O^T += V^T P^T V^T by transposing LDS reads; a lane's outputs belong to the same row: rescaling is lane-local, and skipped
//                  while no maximum of the wave moves.
// Two workgroups share a CU, so that one's exponentials run beside the other's products.
#define PAT_NW 4
#define PAT_BK 64
template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(PAT_NW * 64, 2) paged_attention_tiles_kernel(PagedAttnParams P) {
    typedef typename vec_of<T>::v8 v8;
    typedef typename vec_of<T>::v4 v4;
    constexpr int EPL = Q8 ? 16 : 8, LPR = D / EPL, RPP = PAT_NW * 64 / LPR, PASSES = PAT_BK / RPP;
    constexpr int BUF = 2 * PAT_BK * D;             // elements: K, then V
    constexpr int QS = D / 16, NB = D / 32, KS = PAT_BK / 16, ROWS = 32 * PAT_NW;
    __shared__ __attribute__((aligned(256))) unsigned char lds[2 * BUF * 2];
    __shared__ int lds_hidden[2][PAT_BK];           // rows of a tile with values that were taken out
    AttnItem I;
    if (!attn_item(P, ROWS, I)) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qc = lane & 31, h = lane >> 5;
    const int k0 = I.split * P.split_len, k1 = I.end < k0 + P.split_len ? I.end : k0 + P.split_len;

    const int wrow = I.row0 + 32 * wave;            // the wave's first row
    int r = wrow + qc;
    const bool live = r < I.rows;
    r = live ? r : I.rows - 1;
    const int token = r / P.group, head = I.kvh * P.group + r - token * P.group;
    int lim = I.past + token;                       // last key this lane's row sees, here
    lim = lim < k1 ? lim : k1 - 1;
    v8 qf[QS];
    {
        const T* qr = (const T*)P.q + head * P.q_head_stride + (size_t)(I.first + token) * P.q_row_stride + 8 * h;
#pragma unroll
        for (int s = 0; s < QS; ++s) qf[s] = *(const v8*)(qr + 16 * s);
    }
    const int lim_of_row0 = I.past + I.row0 / P.group;
    int wlast = wrow + 31 < I.rows ? wrow + 31 : I.rows - 1;
    int lim_lo = I.past + wrow / P.group, lim_hi = I.past + wlast / P.group;
    lim_lo = wrow < I.rows ? (lim_lo < k1 ? lim_lo : k1 - 1) : -1;      // a wave without rows only helps to fetch
    lim_hi = wrow < I.rows ? (lim_hi < k1 ? lim_hi : k1 - 1) : -1;

    float m_run = -INFINITY, l_run = 0.f;
    floatx16 o_acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o_acc[i] = floatx16{};

    // Rows lie in LDS one behind the other, their 16-byte chunks in an order that depends on the row: chunk c of row r is at
    // place c ^ order(r).  The reads of K (one chunk of 16 consecutive rows) and the transposing reads of V (four chunks of four
    // consecutive rows) then touch every bank once, and rows can be fetched by loads that write LDS themselves.
    auto k_order = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    auto v_order = [](int r) { return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3); };
    const int lim0 = lim_of_row0 < k1 ? lim_of_row0 : k1 - 1;           // keys up to here are seen by every row of the workgroup
    const int lrow = lane / LPR, lcol = lane % LPR;
    // A wave's rows of a pass lie in one 16-row block, so in one page: its entry is uniform, the rows one behind the other.  Pages of
    // a tile's length or more hold all passes' rows: one look-up a tile instead of one a pass (60 scalar instructions of a tile's
    // 600 or so).
    constexpr int RPW = 64 / LPR;
    const bool whole = P.map.shift >= 6;
    int pg[PASSES];
    auto pages = [&](int key0) {
        pg[0] = page_entry(P.map, I.seq, (key0 + wave * RPW) >> P.map.shift);
        if (!whole) {
#pragma unroll
            for (int i = 1; i < PASSES; ++i) pg[i] = page_entry(P.map, I.seq, (key0 + i * RPP + wave * RPW) >> P.map.shift);
        }
    };
    auto rows_of = [&](int key0, size_t (&row)[PASSES]) {   // takes the entries, and asks for those of the next tile first: loads end in order
        row[0] = stored_row(P, check_page(P.map, pg[0]), I.kvh, key0 + wave * RPW);
#pragma unroll
        for (int i = 1; i < PASSES; ++i) row[i] = row[0] + i * RPP;
        if (!whole) {
#pragma unroll
            for (int i = 1; i < PASSES; ++i) row[i] = stored_row(P, check_page(P.map, pg[i]), I.kvh, key0 + i * RPP + wave * RPW);
        }
        pages(key0 + PAT_BK);
    };
    // values of V that are not finite, in a tile that some row does not see all of: staged as 0, and their rows noted
    auto note = [&](int which, int rr, bool bad) {
        const uint64_t lanes = __ballot(bad);
        if (lcol == 0) lds_hidden[which][rr] = (lanes >> (lane & ~(LPR - 1))) & ((1ull << LPR) - 1) ? 1 : 0;
    };
    // e4m3: through registers, which widen
    u32x4 kr[PASSES], vr[PASSES];
    uint32_t ksr[PASSES], vsr[PASSES];
    auto load_codes = [&](int key0) {
        size_t row[PASSES];
        rows_of(key0, row);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            kr[i] = *(const u32x4*)((const uint8_t*)P.k + row[i] * D + lane * 16);
            vr[i] = *(const u32x4*)((const uint8_t*)P.v + row[i] * D + lane * 16);
            ksr[i] = (P.ks + row[i])[lrow];
            vsr[i] = (P.vs + row[i])[lrow];
        }
    };
    auto stage_codes = [&](int key0, int which) {
        T *bk = (T*)lds + which * BUF, *bv = bk + PAT_BK * D;
        const bool masked = key0 + PAT_BK - 1 > lim0;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int rr = i * RPP + wave * RPW + lrow;
            if (masked && key0 + rr >= k1) { vr[i] = u32x4{0, 0, 0, 0}; vsr[i] = 127; }      // rows behind the end hold anything
            v8 lo, hi;
            e4m3_expand<T>(kr[i], e4m3_scale(ksr[i]), lo, hi);
            *(v8*)(bk + rr * D + 8 * ((2 * lcol) ^ k_order(rr))) = lo;
            *(v8*)(bk + rr * D + 8 * ((2 * lcol + 1) ^ k_order(rr))) = hi;
            e4m3_expand<T>(vr[i], e4m3_scale(vsr[i]), lo, hi);
            if (masked) note(which, rr, take_nonfinite<T>(lo) | take_nonfinite<T>(hi));
            *(v8*)(bv + rr * D + 8 * ((2 * lcol) ^ v_order(rr))) = lo;
            *(v8*)(bv + rr * D + 8 * ((2 * lcol + 1) ^ v_order(rr))) = hi;
        }
    };
    // 16-bit rows: straight into LDS, a lane's place fixed, so the lane fetches the chunk that belongs there
    auto fetch = [&](int key0, int which) {
        size_t row[PASSES];
        rows_of(key0, row);
        const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds + which * (BUF * 2);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r0 = i * RPP + wave * RPW, rr = r0 + lrow;
            const uint32_t from = lrow * (2 * D);
            load_to_lds((const uint8_t*)P.k + row[i] * (2 * D), from + 16 * (lcol ^ k_order(rr)), base + r0 * (2 * D));
            load_to_lds((const uint8_t*)P.v + row[i] * (2 * D), from + 16 * (lcol ^ v_order(rr)), base + (PAT_BK + r0) * (2 * D));
        }
    };
    auto clean = [&](int key0, int which) {         // a fetched tile that some row does not see all of
        T* bv = (T*)lds + which * BUF + PAT_BK * D;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int rr = i * RPP + wave * RPW + lrow;
            v8* at = (v8*)(bv + rr * D + 8 * lcol);
            v8 w = *at;
            const bool behind = key0 + rr >= k1;    // rows behind the end hold anything
            if (behind) w = v8{};
            const bool bad = take_nonfinite<T>(w);
            if (behind | bad) *at = w;
            note(which, rr, bad);
        }
        __syncthreads();
    };
    auto compute = [&](int key0, int which, bool masked) {
        const T *bk = (const T*)lds + which * BUF, *bv = bk + PAT_BK * D;
        __builtin_amdgcn_s_setprio(1);              // over the other workgroup's wave, which has its exponentials to do meanwhile
        floatx16 s_acc[2] = {};
        {
            auto k_frag = [&](int b, int s) { return *(const v8*)(bk + (32 * b + qc) * D + 8 * ((2 * s + h) ^ k_order(qc))); };
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int s = 0; s < QS; ++s) s_acc[b] = mfma32<T>(k_frag(b, s), qf[s], s_acc[b]);
            // LDS reads run four products ahead: left alone, each is issued next to the product that waits for it
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < 2 * QS - 4; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (masked) {
            int seen = lim - key0 - 4 * h;          // opaque, or the 32 differences to it are kept in registers over the whole loop
            asm("" : "+v"(seen));
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s_acc[b][i] = 32 * b + 8 * (i >> 2) + (i & 3) <= seen ? s_acc[b][i] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s_acc[b][i]);
        {
            unsigned a = __builtin_bit_cast(unsigned, mx), c = a;
            lane_swap32(a, c);
            mx = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, c));
        }
        const float m_new = fmaxf(m_run, mx * P.scale_log2e);
        if (__any(m_new > m_run + 8.0f)) {
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
            l_run *= alpha;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) o_acc[b][i] *= alpha;
            m_run = m_new;
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        v8 pf[KS];
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s_acc[b][i], P.scale_log2e, -m_use));
                sum += p;
                pf[2 * b + (i >> 3)][i & 7] = (T)p;
            }
        l_run += sum;
        // slot (h, j) of step ks is key 16 ks + 8 (j >> 2) + 4 h + (j & 3): the order the weights stand in
        auto v_frag = [&](int ks, int b) {
            const int r = 4 * h + ((lane & 15) >> 2), c = 4 * b + ((lane >> 3) & 2) + ((lane & 3) >> 1);      // order(16 ks + r) = order(r)
            const T* a = bv + 16 * ks * D + 4 * (lane & 1);
            const u32x2 lo = read_transposed(a + r * D + 8 * (c ^ v_order(r))), hi = read_transposed(a + (r + 8) * D + 8 * (c ^ v_order(r + 8)));
            return __builtin_bit_cast(v8, u32x4{lo[0], lo[1], hi[0], hi[1]});
        };
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < NB; ++b) o_acc[b] = mfma32<T>(v_frag(ks, b), pf[ks], o_acc[b]);
        if (key0 + PAT_BK - 1 <= lim0) return;
        uint64_t hidden = __ballot(lds_hidden[which][lane] != 0);
        while (hidden) {                            // wave-uniform, and hardly ever entered
            const int key = key0 + __builtin_ctzll(hidden);
            hidden &= hidden - 1;
            const size_t row = stored_row(P, check_page(P.map, page_entry(P.map, I.seq, key >> P.map.shift)), I.kvh, key);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x[4];
                    hidden4<T, D, Q8>(P, row, 32 * b + 8 * i + 4 * h, x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o_acc[b][4 * i + j] += key <= lim ? x[j] : 0.f;
                }
        }
    };

    if (k0 < k1) {
        pages(k0);
        if constexpr (Q8) { load_codes(k0); stage_codes(k0, 0); }
        else fetch(k0, 0);
    }
#pragma unroll
    for (int s = 0; s < QS; ++s) arrived(qf[s]);
    int cur = 0;
    for (int key0 = k0; key0 < k1; key0 += PAT_BK, cur ^= 1) {
        if constexpr (!Q8) loads_done();
        __syncthreads();
        const int nxt = key0 + PAT_BK;
        if constexpr (Q8) {
            if (nxt < k1) load_codes(nxt);
        } else {
            if (key0 + PAT_BK - 1 > lim0) clean(key0, cur);
            if (nxt < k1) fetch(nxt, cur ^ 1);
        }
        if (key0 <= lim_hi) compute(key0, cur, key0 + PAT_BK - 1 > lim_lo);
        if constexpr (Q8) {
            if (nxt < k1) stage_codes(nxt, cur ^ 1);
        }
    }

    {
        unsigned a = __builtin_bit_cast(unsigned, l_run), c = a;
        lane_swap32(a, c);
        l_run = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, c);
    }
    if (!live) return;
    if (I.n_parts <= 1) {
        const float inv = l_run != 0.f ? 1.0f / l_run : 0.f;        // a row that sees nothing: zeros
        T* dst = (T*)P.out + (size_t)(I.first + token) * P.out_stride + (size_t)head * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (T)(o_acc[b][4 * i + j] * inv);
                *(v4*)(dst + 32 * b + 8 * i) = w;
            }
    } else {
        const size_t pr = ((size_t)I.split * P.n_rows + I.first + token) * P.n_heads + head;
        float* dst = P.part_o + pr * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                floatx4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = o_acc[b][4 * i + j];
                *(floatx4*)(dst + 32 * b + 8 * i) = w;
            }
        if (h == 0) { P.part_ml[pr * 2] = m_run; P.part_ml[pr * 2 + 1] = l_run; }
    }
}

// Joins the parts of the key axis: one workgroup a (row, head); each of its waves takes every fourth part, four of them in
// flight at once.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(PagedAttnParams P, int tile_rows) {
    constexpr int E = D / 64, MAX = 4;                      // outputs a lane, parts a wave at a time
    typedef float vecE __attribute__((ext_vector_type(E)));
    __shared__ float acc[4][D];
    const int t = blockIdx.x / P.n_heads, head = blockIdx.x % P.n_heads, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const size_t step = (size_t)P.n_rows * P.n_heads, row = (size_t)t * P.n_heads + head;
    const bool there = lane < P.n_splits;                   // loaded before it is known how many parts the row has
    float m = there ? P.part_ml[(row + lane * step) * 2] : -INFINITY, l = there ? P.part_ml[(row + lane * step) * 2 + 1] : 0.f;
    const int seq = seq_of_row(P.cu_rows, P.n_seqs, t);
    if (seq >= P.n_seqs) return;
    const int first = P.cu_rows[seq], rows = (P.cu_rows[seq + 1] - first) * P.group, past = P.seq_lens[seq];
    const int r = (t - first) * P.group + head % P.group;
    const int parts = __builtin_amdgcn_readfirstlane((attn_tile_end(P, past, rows, r / tile_rows, tile_rows) + P.split_len - 1) / P.split_len);
    if (parts <= 1) return;                                 // written already
    if (lane >= parts) { m = -INFINITY; l = 0.f; }
    const float top = wave_max_f32_dpp(m);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);       // 0 in the lanes behind the last part
    const float sum = wave_sum_f32_dpp(l * f);
    vecE mine = {};
    for (int s0 = wave; s0 < parts; s0 += 4 * MAX) {
        vecE o[MAX];
#pragma unroll
        for (int i = 0; i < MAX; ++i) {
            const int s = s0 + 4 * i < parts ? s0 + 4 * i : s0;                   // no branch: all of them are in flight
            o[i] = *(const vecE*)(P.part_o + (row + s * step) * D + lane * E);
        }
#pragma unroll
        for (int i = 0; i < MAX; ++i) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), (s0 + 4 * i) & 63));
            mine += o[i] * (s0 + 4 * i < parts ? w : 0.f);
        }
    }
    *(vecE*)&acc[wave][lane * E] = mine;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += 256) {
        const float inv = sum != 0.f ? 1.0f / sum : 0.f;
        ((T*)P.out)[(size_t)t * P.out_stride + (size_t)head * D + d] = (T)(((acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d])) * inv);
    }
}

struct AttnPlan { int tile_rows, n_tiles, n_splits, split_len; };

static AttnPlan attn_plan(int n_seqs, int max_rows, int max_len, int n_heads, int h_kv) {
    AttnPlan A;
    const int rows = max_rows * (n_heads / h_kv);
    A.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 128;
    A.n_tiles = (rows + A.tile_rows - 1) / A.tile_rows;
    const int64_t base = (int64_t)n_seqs * h_kv * A.n_tiles;
    int64_t want = (2048 + base - 1) / base;
    want = want > 64 ? 64 : want;
    int64_t len = (max_len + want - 1) / want;
    len = len < 256 ? 256 : len;
    A.split_len = (int)((len + 127) / 128 * 128);
    A.n_splits = (max_len + A.split_len - 1) / A.split_len;
    if (A.n_splits < 1) A.n_splits = 1;
    return A;
}

extern "C" size_t sq_paged_attention_workspace_bytes(int n_seqs, int n_rows, int max_rows, int max_len, int n_heads, int h_kv, int d) {
    if (n_seqs <= 0 || n_rows <= 0 || max_rows <= 0 || max_len <= 0 || n_heads <= 0 || h_kv <= 0 || n_heads % h_kv || d <= 0) return 0;
    if (max_rows > n_rows) max_rows = n_rows;
    const AttnPlan A = attn_plan(n_seqs, max_rows, max_len, n_heads, h_kv);
    return A.n_splits > 1 ? (size_t)A.n_splits * n_rows * n_heads * (d + 2) * sizeof(float) : 0;
}

extern "C" int sq_paged_attention(const void* q, int64_t q_head_stride, int64_t q_row_stride, const void* k_pages, const void* v_pages,
                                  const void* k_scales, const void* v_scales, void* out, int64_t out_stride,
                                  const int32_t* d_page_table, int table_width, int n_pages, int page_size, const int32_t* d_seq_lens,
                                  const int32_t* d_cu_rows, int n_seqs, int n_rows, int max_rows, int max_len, int n_heads, int h_kv,
                                  int d, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (n_seqs < 0 || n_rows < 0 || max_rows < 0 || max_len < 0 || n_heads <= 0 || h_kv <= 0 || n_heads % h_kv || table_width < 0 || n_pages <= 0)
        return SQ_EINVAL;
    if (!k_scales != !v_scales || !(scale > 0.f) || !(scale < INFINITY)) return SQ_EINVAL;
    const int shift = page_shift(page_size);
    if ((d != 64 && d != 128) || shift < 0 || (dtype != SQ_DTYPE_F16 && dtype != SQ_DTYPE_BF16)) return SQ_EUNSUPPORTED;
    if (n_rows == 0 || n_seqs == 0 || max_rows == 0) return SQ_OK;
    if (max_len < 1 || (int64_t)max_len > ((int64_t)table_width << shift)) return SQ_EINVAL;
    if (!q || !k_pages || !v_pages || !out || !d_page_table || !d_seq_lens || !d_cu_rows) return SQ_EINVAL;
    if ((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) || ((uintptr_t)out & 7) || ((q_head_stride | q_row_stride) & 7) || (out_stride & 3))
        return SQ_EINVAL;
    if (max_rows > n_rows) max_rows = n_rows;
    const AttnPlan A = attn_plan(n_seqs, max_rows, max_len, n_heads, h_kv);
    const size_t need = sq_paged_attention_workspace_bytes(n_seqs, n_rows, max_rows, max_len, n_heads, h_kv, d);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return SQ_EINVAL;
    const int64_t grid = (int64_t)n_seqs * h_kv * A.n_tiles * A.n_splits, join = (int64_t)n_rows * n_heads;
    if (grid > 0x7fffffff || join > 0x7fffffff) return SQ_EUNSUPPORTED;
    PagedAttnParams P = {q, q_head_stride, q_row_stride, k_pages, v_pages, (const uint8_t*)k_scales, (const uint8_t*)v_scales, out, out_stride,
                         {d_page_table, table_width, n_pages, shift}, d_seq_lens, d_cu_rows, n_seqs, n_rows, n_heads, h_kv, n_heads / h_kv,
                         scale * 1.4426950408889634f, max_len, A.n_tiles, A.n_splits, A.split_len, (float*)workspace,
                         need ? (float*)workspace + (size_t)A.n_splits * n_rows * n_heads * d : nullptr};
    hipStream_t st = (hipStream_t)stream;
#define SQ_A(TT, DD, QQ, MM) hipLaunchKernelGGL((paged_attention_rows_kernel<TT, DD, QQ, MM>), dim3((unsigned)grid), dim3(PAD_NW * 64), 0, st, P)
#define SQ_AT(TT, DD, QQ) hipLaunchKernelGGL((paged_attention_tiles_kernel<TT, DD, QQ>), dim3((unsigned)grid), dim3(PAT_NW * 64), 0, st, P)
#define SQ_AM(TT, DD, QQ) do { if (A.tile_rows == 16) SQ_A(TT, DD, QQ, 1); else if (A.tile_rows == 32) SQ_A(TT, DD, QQ, 2); else SQ_AT(TT, DD, QQ); } while (0)
#define SQ_AD(TT, DD) do { if (k_scales) SQ_AM(TT, DD, true); else SQ_AM(TT, DD, false); } while (0)
    if (dtype == SQ_DTYPE_F16) { if (d == 128) SQ_AD(half_t, 128); else SQ_AD(half_t, 64); }
    else                       { if (d == 128) SQ_AD(bf16_t, 128); else SQ_AD(bf16_t, 64); }
#undef SQ_AD
#undef SQ_AM
#undef SQ_AT
#undef SQ_A
    int rc = sq_check_launch();
    if (rc != SQ_OK || A.n_splits <= 1) return rc;
#define SQ_J(TT, DD) hipLaunchKernelGGL((paged_attention_join_kernel<TT, DD>), dim3((unsigned)join), dim3(256), 0, st, P, A.tile_rows)
    if (dtype == SQ_DTYPE_F16) { if (d == 128) SQ_J(half_t, 128); else SQ_J(half_t, 64); }
    else                       { if (d == 128) SQ_J(bf16_t, 128); else SQ_J(bf16_t, 64); }
#undef SQ_J
    return sq_check_launch();
}
