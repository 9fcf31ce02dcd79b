// Attention of a ragged batch's new tokens over a paged KV cache (their own rows already written): for sequence b with `past`
// stored rows and n new ones, row i attends keys [0, past + i],
//     o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale * q . k_j,
// in one pass over the keys with a running maximum and sum in fp32.  Weights are rounded to the element type once, because the matrix
// instructions take both operands of the second product so, and the sum is taken of the rounded ones: a result is off by at most half a
// step of the type times sum_j w_j |v_j - o|, beside half a step of its own.  The query heads that share a KV head are packed into the
// same rows of a tile (row r = token r / group, head r % group), so that every stored row is read once for all of them.
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
    int n_tiles, n_splits, split_len;      // tiles: row tiles a (sequence, KV head), parts of the key axis, keys a part
    int tile_rows, n_groups;               // rows: workgroups that share the keys of all units; 0: one a unit
    float* part_o;                         // unnormalised sums.  tiles: [n_splits][n_rows * n_heads][D]; rows: [2 * n_groups][rows a tile][D]
    float* part_ml;                        // [..][2]: maximum (log2 units), sum
    int2* units;                           // rows: [n_seqs * h_kv] {place of the first part, parts}
};

template <typename T> __device__ __forceinline__ floatx4 mfma16(typename vec_of<T>::v8 a, typename vec_of<T>::v8 b, floatx4 c) {
    if constexpr (__is_same(T, half_t)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <typename T> __device__ __forceinline__ floatx16 mfma32(typename vec_of<T>::v8 a, typename vec_of<T>::v8 b, floatx16 c) {
    if constexpr (__is_same(T, half_t)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// c + a[0] + a[1] + .. of a fragment's eight weights.  What the second product uses is what the sum is taken of, so that a weight's
// rounding is one of the whole row's scale where that weight is most of the row, and not of the result.
template <typename T> __device__ __forceinline__ float add_weights(typename vec_of<T>::v8 a, float c) {
    typedef typename vec_of<T>::v2 v2;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const v2 two = {a[i], a[i + 1]}, one = {(T)1.f, (T)1.f};
        float& to = i & 2 ? d : c;
        if constexpr (__is_same(T, half_t)) to = __builtin_amdgcn_fdot2(two, one, to, false);
        else to = __builtin_amdgcn_fdot2_f32_bf16(two, one, to, false);
    }
    return c + d;
}

// log2 of what weights are multiplied by before they are rounded for the second product, numerator and denominator alike, with
// `headroom` doublings left: fp16 ends at 2^16 and loses bits below 2^-14.  From 1 down, the weights of a long context under one key
// that stands out would be among those: 100000 of e^-17 are a 250th of the row, and each of them less than half of the smallest step.
template <typename T> constexpr float weight_shift(int headroom) { return __is_same(T, half_t) ? (float)(15 - headroom) : 0.f; }

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
    if constexpr (Q8) {                             // (a code that is NaN, or one whose value T does not hold)
        const uint32_t code = *(const uint32_t*)((const uint8_t*)P.v + row * D + d);
        typename vec_of<T>::v8 w, none;
        e4m3_expand<T>(u32x4{code, 0, 0, 0}, e4m3_scale(P.vs[row]), w, none);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __builtin_fabsf((float)w[j]) < INFINITY ? 0.f : (float)w[j];
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
// stored rows of sequence b, no more than the keys that count: a length of any size (a padding's marker) overflows nothing
__device__ __forceinline__ int past_of(const PagedAttnParams& P, int length) { return length < P.max_len ? length : P.max_len; }
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
    I.past = past_of(P, __builtin_amdgcn_readfirstlane(P.seq_lens[I.seq]));
    if (I.first < 0 || n <= 0 || n > P.n_rows - I.first) return false;      // no rows, or offsets that name none
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

// Few rows (a decoding step, a drafted chunk): bound by the bytes of K and V.  Four waves walk the 32-key chunks of a unit -- a
// (sequence, KV head) pair -- in turn, each with its own running softmax, and join through LDS.  Per chunk
//   S^T = K Q^T    A = K rows, B = Q: a lane holds 8 scores of one query row, in the order the second product wants them
//   O^T += V^T P^T A = V^T by transposing LDS reads, B = P^T straight from the registers S^T left behind.
// Both come as whole rows, 16 bytes a lane, past the caches (nothing reads them again before much else has passed through), and
// go through the wave's own LDS.  Measured with 48 sequences of 300-6000 e4m3 keys | 16 chunks of 1-7 drafted rows, fp16: cached
// loads 72 | 52 us; K straight into its product's registers, a quarter of a row a lane, cached beside uncached V 66 | 48 us,
// uncached 64 | 60 us; this 64 | 46 us.
// The keys of all units, in order, are shared out evenly over the workgroups that fit the card, in steps of 128: a workgroup takes
// the end of one unit, whole ones, and the beginning of another, and leaves the sums of the first and the last for the join;
// whatever the lengths, all of them end together.  The next chunk's rows are asked for as soon as this one's have left their
// registers, the next unit's first ones too: it is looked up when this one begins.  (Two workgroups a CU: three read 10 % slower.)
// Sequences of few hundred keys pay for the waves' joins: 2048 of 50-300 keys, 64 / 8 heads, fp16, 437 us (3.4 TB/s), 512 of 100-900
// 213 us (4.8), 200 of 1000-3000 285 us (6.0).
#define PAD_NW 4
#define PAD_BK 32
#define PAD_STEP (PAD_NW * PAD_BK)

// the packed rows of sequence b, their first row, stored rows and key end; offsets that name no rows: none
struct Rows { int first, rows, past, end; };
// UNIFORM: by the scalar unit, so that no vector load in flight is waited for
template <bool UNIFORM = false> __device__ __forceinline__ Rows rows_of_seq(const PagedAttnParams& P, int b) {
    typedef const __attribute__((address_space(4))) int32_t* scalar;
    Rows R;
    int upto;
    if constexpr (UNIFORM) {
        const scalar cu = (scalar)(uintptr_t)(P.cu_rows + b), lens = (scalar)(uintptr_t)(P.seq_lens + b);
        R.first = cu[0]; upto = cu[1]; R.past = lens[0];
    } else {
        R.first = P.cu_rows[b]; upto = P.cu_rows[b + 1]; R.past = P.seq_lens[b];
    }
    R.past = past_of(P, R.past);
    const int n = upto - R.first;
    R.rows = R.first >= 0 && n > 0 && n <= P.n_rows - R.first ? n * P.group : 0;
    R.end = R.rows ? attn_tile_end(P, R.past, R.rows, 0, P.tile_rows) : 0;
    return R;
}
__device__ __forceinline__ int steps_of(int end) { return (end + PAD_STEP - 1) / PAD_STEP; }

// By one wave: the sequence that step `group * per` of all belongs to (n_seqs: none), the step's place among the sequence's (KV
// heads one behind the other), and per, the steps a workgroup.  The host has seen to it that all steps' number fits 31 bits.
__device__ __forceinline__ int share(const PagedAttnParams& P, int group, int& per, int& place) {
    const int lane = threadIdx.x & 63;
    int mine = lane < P.n_seqs ? steps_of(rows_of_seq(P, lane).end) : 0;
    uint32_t total = wave_sum_u32_dpp(mine);
    for (int base = 64; base < P.n_seqs; base += 64)
        total += wave_sum_u32_dpp(base + lane < P.n_seqs ? steps_of(rows_of_seq(P, base + lane).end) : 0);
    const uint32_t all = total * (uint32_t)P.h_kv, even = (all + P.n_groups - 1) / (uint32_t)P.n_groups;
    per = even > 2 ? (int)even : 2;                         // a part of fewer keys costs more to join than to walk
    const uint32_t at = (uint32_t)group * (uint32_t)per;
    if (at >= all) return P.n_seqs;
    uint32_t before = 0;
    for (int base = 0; base < P.n_seqs; base += 64) {
        if (base) mine = base + lane < P.n_seqs ? steps_of(rows_of_seq(P, base + lane).end) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int w = __shfl_up(upto, o, 64); if (lane >= o) upto += w; }
        const uint64_t hit = __ballot((before + (uint32_t)upto) * (uint32_t)P.h_kv > at);
        if (hit) {
            const int j = __builtin_ctzll(hit);
            before += __builtin_amdgcn_readlane(upto, j) - __builtin_amdgcn_readlane(mine, j);
            place = (int)(at - before * (uint32_t)P.h_kv);
            return base + j;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return P.n_seqs;
}

template <typename T, int D, bool Q8, int MT>
__global__ void __launch_bounds__(PAD_NW * 64, 2) paged_attention_rows_kernel(PagedAttnParams P) {
    typedef typename vec_of<T>::v8 v8;
    typedef typename vec_of<T>::v4 v4;
    constexpr int ESZ = Q8 ? 1 : 2, LPR = D * ESZ / 16, RPP = 64 / LPR, PASSES = PAD_BK / RPP;   // lanes a row, rows a pass
    constexpr int DSTEPS = D / 32, NT = D / 16, ROWS = 16 * MT;
    constexpr int KSTR = D + 8, VSTR = D + 16;      // 16-byte reads of 16 rows, 8-byte transposing reads of 8 rows: all banks once
    constexpr int WAVE_BYTES = PAD_BK * (KSTR + VSTR) * 2, OSTR = D + 4;
    constexpr int LDS_BYTES = PAD_NW * (WAVE_BYTES > ROWS * OSTR * 4 ? WAVE_BYTES : ROWS * OSTR * 4);
    __shared__ __attribute__((aligned(16))) unsigned char lds[LDS_BYTES];
    __shared__ float lds_ml[PAD_NW][ROWS][2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qc = lane & 15, g = lane >> 4;
    const int lrow = lane / LPR, lcol = lane % LPR;
    T *my_k = (T*)(lds + wave * WAVE_BYTES), *my_v = my_k + PAD_BK * KSTR;

    // ---- where it is: all of this in scalar registers, so that what branches on it is uniform ----
    int seq, kvh, from = 0, left = 0x7fffffff, per = 0;     // from: the step of the unit to begin with; left: steps still to do
    if (P.n_groups) {
        int place = 0;
        seq = __builtin_amdgcn_readfirstlane(share(P, blockIdx.x, per, place));
        if (seq >= P.n_seqs) return;
        left = per = __builtin_amdgcn_readfirstlane(per);
        from = __builtin_amdgcn_readfirstlane(place);
    } else {
        seq = blockIdx.x / P.h_kv;
    }
    auto at_seq = [&](int b, Rows& r) {             // -> the steps of one of its units
        r = rows_of_seq<true>(P, b);
        r.rows = r.rows < ROWS ? r.rows : ROWS;
        return steps_of(r.end);
    };
    Rows R;
    int steps = at_seq(seq, R), upto, k0, k1;
    auto at_unit = [&]() {
        upto = left < steps - from ? from + left : steps;
        k0 = from * PAD_STEP;
        k1 = R.end < upto * PAD_STEP ? R.end : upto * PAD_STEP;
    };
    if (P.n_groups) {
        kvh = from / steps;
        from -= kvh * steps;
    } else {
        kvh = blockIdx.x - seq * P.h_kv;
        if (R.rows == 0) return;
    }
    at_unit();

    // ---- loads ----
    u32x4 kr[PASSES], vr[PASSES];
    uint32_t ksr[PASSES], vsr[PASSES];
    size_t row[2];                                  // scalar: first rows of the chunk's halves
    int ea = 0, eb = 0;                             // entries of the pages that hold the halves of the next chunk
    int na = 0, nb = 0;                             // of the next unit's first one
    v8 qf[MT][DSTEPS];
    int lim[MT];                                    // last key this lane's query row sees, here
    auto pages = [&](int of_seq, int key0, int& a, int& b) {
        a = page_entry(P.map, of_seq, key0 >> P.map.shift);
        b = page_entry(P.map, of_seq, (key0 + 16) >> P.map.shift);
    };
    auto take = [&](int of_kvh, int key0, int a, int b) {
        row[0] = stored_row(P, check_page(P.map, a), of_kvh, key0);
        row[1] = stored_row(P, check_page(P.map, b), of_kvh, key0 + 16);
    };
    auto load = [&]() {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const size_t r = i * RPP < 16 ? row[0] + i * RPP : row[1] + (i * RPP - 16);
            const uint32_t at = (uint32_t)lane * 16;                    // rows lie one behind the other
            kr[i] = __builtin_nontemporal_load((const u32x4*)((const uint8_t*)P.k + r * (D * ESZ) + at));
            vr[i] = __builtin_nontemporal_load((const u32x4*)((const uint8_t*)P.v + r * (D * ESZ) + at));
            if constexpr (Q8) { ksr[i] = (P.ks + r)[lrow]; vsr[i] = (P.vs + r)[lrow]; }
        }
    };
    auto load_q = [&]() {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            int r = 16 * mt + qc;
            r = r < R.rows ? r : R.rows - 1;
            const int token = r / P.group, head = kvh * P.group + r - token * P.group;
            lim[mt] = R.past + token < k1 ? R.past + token : k1 - 1;
            const T* qr = (const T*)P.q + head * P.q_head_stride + (size_t)(R.first + token) * P.q_row_stride + 8 * g;
#pragma unroll
            for (int s = 0; s < DSTEPS; ++s) qf[mt][s] = *(const v8*)(qr + 32 * s);
        }
    };
    {
        int fa, fb;
        pages(seq, k0 + wave * PAD_BK, fa, fb);
        pages(seq, k0 + wave * PAD_BK + PAD_STEP, ea, eb);
        take(kvh, k0 + wave * PAD_BK, fa, fb);      // (a wave without a chunk here loads one all the same, in bounds)
        load();
        load_q();
    }

    for (bool first_unit = true;; first_unit = false) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < DSTEPS; ++s) arrived(qf[mt][s]);
        // the next unit, looked up while this one's first rows are on their way: its own first rows follow this one's last
        int nseq = seq, nkvh = kvh + 1, nsteps = steps;
        Rows nR = R;
        bool next = P.n_groups && left > upto - from;
        if (next && nkvh == P.h_kv) {
            nkvh = 0;
            do ++nseq; while (nseq < P.n_seqs && (nsteps = at_seq(nseq, nR)) == 0);
            next = nseq < P.n_seqs;
        }
        if (next) pages(nseq, wave * PAD_BK, na, nb);
        const int lim0 = R.past;                    // keys up to here are seen by every row
        float m_run[MT], l_run[MT];
        floatx4 o_acc[MT][NT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m_run[mt] = -INFINITY; l_run[mt] = 0.f;
#pragma unroll
            for (int i = 0; i < NT; ++i) o_acc[mt][i] = floatx4{0.f, 0.f, 0.f, 0.f};
        }

        for (int key0 = k0 + wave * PAD_BK; key0 < k1; key0 += PAD_STEP) {
            const bool tail = key0 + PAD_BK > k1;   // rows behind the end hold anything: their weights are 0, and so are they
            const bool masked = tail || key0 + PAD_BK - 1 > lim0, more = key0 + PAD_STEP < k1;
            uint32_t hidden = 0;                    // rows of the chunk with values that were taken out
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int rr = i * RPP + lrow;
                bool bad = false;
                if (tail && key0 + rr >= k1) { vr[i] = u32x4{0, 0, 0, 0}; if constexpr (Q8) vsr[i] = 127; }
                if constexpr (Q8) {
                    v8 lo, hi;
                    e4m3_expand<T>(kr[i], e4m3_scale(ksr[i]), lo, hi);
                    *(v8*)(my_k + rr * KSTR + 16 * lcol) = lo;
                    *(v8*)(my_k + rr * KSTR + 16 * lcol + 8) = hi;
                    e4m3_expand<T>(vr[i], e4m3_scale(vsr[i]), lo, hi);
                    if (masked) bad = take_nonfinite<T>(lo) | take_nonfinite<T>(hi);
                    *(v8*)(my_v + rr * VSTR + 16 * lcol) = lo;
                    *(v8*)(my_v + rr * VSTR + 16 * lcol + 8) = hi;
                } else {
                    *(u32x4*)(my_k + rr * KSTR + 8 * lcol) = kr[i];
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
            {                                       // the entries of the chunk after the next come first: loads end in order
                const int key = more ? key0 + PAD_STEP : wave * PAD_BK;
                take(more ? kvh : nkvh, key, more ? ea : na, more ? eb : nb);
                pages(more || !next ? seq : nseq, key + PAD_STEP, ea, eb);
                if (more || next) load();
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
                    int seen = lim[mt] - key0 - 4 * g;      // opaque: not eight differences kept over the loop
                    asm("" : "+v"(seen));
#pragma unroll
                    for (int j = 0; j < 8; ++j) sv[j] = 16 * (j >> 2) + (j & 3) <= seen ? sv[j] : -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) cmax = fmaxf(cmax, sv[j]);
                cmax = group4_max(cmax);
                const float m_new = fmaxf(m_run[mt], cmax);
                const float m_fin = m_new == -INFINITY ? 0.f : m_new;       // nothing seen so far
                if (__any(m_new > m_run[mt])) {
                    const float alpha = __builtin_amdgcn_exp2f(m_run[mt] - m_fin);
                    l_run[mt] *= alpha;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o_acc[mt][nt] *= alpha;
                    m_run[mt] = m_new;
                }
                const float m_use = m_fin - weight_shift<T>(0);
#pragma unroll
                for (int j = 0; j < 8; ++j) pf[mt][j] = (T)__builtin_amdgcn_exp2f(sv[j] - m_use);
                l_run[mt] = add_weights<T>(pf[mt], l_run[mt]);
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
            while (hidden) {                        // wave-uniform, and hardly ever entered
                const int key = key0 + __builtin_ctz(hidden);
                hidden &= hidden - 1;
                const size_t at = stored_row(P, check_page(P.map, page_entry(P.map, seq, key >> P.map.shift)), kvh, key);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[4];
                    hidden4<T, D, Q8>(P, at, 16 * nt + 4 * g, x);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o_acc[mt][nt][j] += key <= lim[mt] ? x[j] : 0.f;
                }
            }
            __builtin_amdgcn_wave_barrier();
        }

        if (next && k0 + wave * PAD_BK >= k1) {     // a wave without a chunk of this unit
            take(nkvh, wave * PAD_BK, na, nb);
            pages(nseq, wave * PAD_BK + PAD_STEP, ea, eb);
            load();
        }

        // ---- join the waves, with the next unit's first rows on their way ----
        const bool whole = from == 0 && upto == steps;
        const int done_rows = R.rows, done_first = R.first, done_head = kvh * P.group;
        if (P.n_groups && from == 0 && tid == 0) {  // where the join finds the unit's parts
            int2* const u = P.units + seq * P.h_kv + kvh;
            *u = int2{(int)(2 * blockIdx.x + (first_unit ? 0 : 1)), whole ? 1 : 1 + (steps - upto + per - 1) / per};
        }
        if (next) {
            left -= upto - from;
            from = 0;
            seq = nseq; kvh = nkvh; steps = nsteps; R = nR;
            at_unit();
        }
        __syncthreads();                            // everyone is done with the staging area
        float* lds_o = (float*)lds;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float l = group4_sum(l_run[mt]);
            if (g == 0) { lds_ml[wave][16 * mt + qc][0] = m_run[mt]; lds_ml[wave][16 * mt + qc][1] = l; }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) *(floatx4*)(lds_o + (wave * ROWS + 16 * mt + qc) * OSTR + 16 * nt + 4 * g) = o_acc[mt][nt];
        }
        __syncthreads();
        if (next) load_q();
        for (int e = tid; e < ROWS * (D / 4); e += PAD_NW * 64) {
            const int r = e / (D / 4), col = 4 * (e % (D / 4));
            if (r >= done_rows) break;              // rows ascend with e
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < PAD_NW; ++w) m = fmaxf(m, lds_ml[w][r][0]);
            floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < PAD_NW; ++w) {
                const float mw = lds_ml[w][r][0], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
                l += lds_ml[w][r][1] * f;
                o += *(const floatx4*)(lds_o + (w * ROWS + r) * OSTR + col) * f;
            }
            if (whole) {
                const int token = r / P.group, head = done_head + r - token * P.group;
                const float inv = l != 0.f ? 1.0f / l : 0.f;        // a row that sees nothing: zeros
                v4 res;
#pragma unroll
                for (int j = 0; j < 4; ++j) res[j] = (T)(o[j] * inv);
                *(v4*)((T*)P.out + (size_t)(done_first + token) * P.out_stride + (size_t)head * D + col) = res;
            } else {
                const size_t pr = (size_t)(2 * blockIdx.x + (first_unit ? 0 : 1)) * ROWS + r;
                *(floatx4*)(P.part_o + pr * D + col) = o;
                if (col == 0) { P.part_ml[pr * 2] = m; P.part_ml[pr * 2 + 1] = l; }
            }
        }
        if (!next) return;
        __syncthreads();                            // the sums have been read: LDS is free again
    }
}

// Many rows (a prompt's chunk, a wide tree of shared heads): bound by the matrix products and the exponentials between them.  A
// workgroup's four waves hold 32 rows each and share 64-key tiles of K and V in LDS (two buffers: the next tile's rows travel
// global -> registers while this one is computed, registers -> LDS behind it; one barrier a tile).  With 32 x 32 products,
//   S^T = K Q^T    leaves a lane with 32 scores of ONE row: its maximum and sum are lane-local but for one exchange between the
//                  two half-waves, and the weights are the second product's B operand where they stand
//   O^T += V^T P^T V^T by transposing LDS reads; a lane's outputs belong to the same row: rescaling is lane-local, and skipped
//                  while no maximum of the wave moves.
// Two workgroups share a CU, so that one's exponentials run beside the other's products.  SHARED: at most a tile of rows a unit, and the
// units' keys are shared out as the rows kernel's are.
// A row's maximum is replaced only when it grows by more than a factor of 2^8: weights then reach 256 instead of 1, with the same
// relative rounding to the element type and the same fp32 sum; what is lost is that the largest weight is no longer exactly 1, and
// the sum of the rounded weights makes up for most of it (error against 64 bits 0.0017; 0.0019 with the sum of the unrounded ones;
// 0.0016 of it is the output's own rounding).  16-bit rows go global -> LDS without registers; e4m3 rows through registers, which widen them.
// 4096 rows of 64 heads behind 4001 stored ones, 8 KV heads of 128, bf16: 771 us, 1.05 PFLOP/s of the products that the mask leaves
// (a large library product here: 1.26).  Of a wave's 2000 or so cycles a tile, 1024 are products; the exponentials and the
// maximum's pass run beside the other wave's products only in part (a priority for one of the two changes nothing; three workgroups
// a CU do not fit the registers).
#define PAT_NW 4
#define PAT_BK 64
template <typename T, int D, bool Q8, bool SHARED>
__global__ void __launch_bounds__(PAT_NW * 64, 2) paged_attention_tiles_kernel(PagedAttnParams P) {
    typedef typename vec_of<T>::v8 v8;
    typedef typename vec_of<T>::v4 v4;
    constexpr int EPL = Q8 ? 16 : 8, LPR = D / EPL, RPP = PAT_NW * 64 / LPR, PASSES = PAT_BK / RPP;
    constexpr int BUF = 2 * PAT_BK * D;             // elements: K, then V
    constexpr int QS = D / 16, NB = D / 32, KS = PAT_BK / 16, ROWS = 32 * PAT_NW;
    __shared__ __attribute__((aligned(256))) unsigned char lds[2 * BUF * 2];
    __shared__ int lds_hidden[2][PAT_BK];           // rows of a tile with values that were taken out
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qc = lane & 31, h = lane >> 5;

    // ---- what it works on; SHARED: a share of all units' keys, as in the rows kernel ----
    AttnItem I;
    int k0, k1, from = 0, left = 0, per = 0, steps = 0, upto = 0;
    auto at_unit = [&]() {
        upto = left < steps - from ? from + left : steps;
        k0 = from * PAD_STEP;
        k1 = I.end < upto * PAD_STEP ? I.end : upto * PAD_STEP;
    };
    if constexpr (SHARED) {
        int place = 0;
        I.seq = __builtin_amdgcn_readfirstlane(share(P, blockIdx.x, per, place));
        if (I.seq >= P.n_seqs) return;
        left = per = __builtin_amdgcn_readfirstlane(per);
        from = __builtin_amdgcn_readfirstlane(place);
        const Rows R = rows_of_seq<true>(P, I.seq);
        I.first = R.first; I.past = R.past; I.end = R.end; I.row0 = 0;
        I.rows = R.rows < P.tile_rows ? R.rows : P.tile_rows;
        steps = steps_of(R.end);
        I.kvh = from / steps;
        from -= I.kvh * steps;
        at_unit();
    } else {
        if (!attn_item(P, ROWS, I)) return;
        k0 = I.split * P.split_len;
        k1 = I.end < k0 + P.split_len ? I.end : k0 + P.split_len;
    }

    // ---- the wave's rows ----
    int r, token, head, lim, lim_lo, lim_hi, lim0;  // lim: last key this lane's row sees, here; lim0: keys up to it are seen by every row of the workgroup
    bool live;
    v8 qf[QS];
    auto enter = [&]() {
        const int wrow = I.row0 + 32 * wave;        // the wave's first row
        r = wrow + qc;
        live = r < I.rows;
        r = live ? r : I.rows - 1;
        token = r / P.group; head = I.kvh * P.group + r - token * P.group;
        lim = I.past + token;
        lim = lim < k1 ? lim : k1 - 1;
        const T* qr = (const T*)P.q + head * P.q_head_stride + (size_t)(I.first + token) * P.q_row_stride + 8 * h;
#pragma unroll
        for (int s = 0; s < QS; ++s) qf[s] = *(const v8*)(qr + 16 * s);
        const int lim_of_row0 = I.past + I.row0 / P.group;
        int wlast = wrow + 31 < I.rows ? wrow + 31 : I.rows - 1;
        lim_lo = I.past + wrow / P.group; lim_hi = I.past + wlast / P.group;
        lim_lo = wrow < I.rows ? (lim_lo < k1 ? lim_lo : k1 - 1) : -1;      // a wave without rows only helps to fetch
        lim_hi = wrow < I.rows ? (lim_hi < k1 ? lim_hi : k1 - 1) : -1;
        lim0 = lim_of_row0 < k1 ? lim_of_row0 : k1 - 1;
    };
    enter();

    float m_run, l_run;
    floatx16 o_acc[NB];

    // Rows lie in LDS one behind the other, their 16-byte chunks in an order that depends on the row: chunk c of row r is at
    // place c ^ order(r).  The reads of K (one chunk of 16 consecutive rows) and the transposing reads of V (four chunks of four
    // consecutive rows) then touch every bank once, and rows can be fetched by loads that write LDS themselves.
    auto k_order = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    auto v_order = [](int r) { return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3); };
    const int lrow = lane / LPR, lcol = lane % LPR;
    // A wave's rows of a pass lie in one 16-row block, so in one page: its entry is uniform, the rows one behind the other.  Pages of
    // a tile's length or more hold all passes' rows: one look-up a tile instead of one a pass (60 scalar instructions of a tile's
    // 600 or so).
    constexpr int RPW = 64 / LPR;
    const bool whole = P.map.shift >= 6;
    int pg[PASSES], npg[PASSES];                    // entries of the next tile; of the next unit's first one
    auto pages = [&](int seq, int key0) {
        pg[0] = page_entry(P.map, seq, (key0 + wave * RPW) >> P.map.shift);
        if (!whole) {
#pragma unroll
            for (int i = 1; i < PASSES; ++i) pg[i] = page_entry(P.map, seq, (key0 + i * RPP + wave * RPW) >> P.map.shift);
        }
    };
    auto rows_of = [&](int seq, int kvh, int key0, const int (&e)[PASSES], size_t (&row)[PASSES]) {   // and asks for the entries of the next tile first: loads end in order
        row[0] = stored_row(P, check_page(P.map, e[0]), kvh, key0 + wave * RPW);
#pragma unroll
        for (int i = 1; i < PASSES; ++i) row[i] = row[0] + i * RPP;
        if (!whole) {
#pragma unroll
            for (int i = 1; i < PASSES; ++i) row[i] = stored_row(P, check_page(P.map, e[i]), kvh, key0 + i * RPP + wave * RPW);
        }
        pages(seq, key0 + PAT_BK);
    };
    // values of V that are not finite, in a tile that some row does not see all of: staged as 0, and their rows noted
    auto note = [&](int which, int rr, bool bad) {
        const uint64_t lanes = __ballot(bad);
        if (lcol == 0) lds_hidden[which][rr] = (lanes >> (lane & ~(LPR - 1))) & ((1ull << LPR) - 1) ? 1 : 0;
    };
    // e4m3: through registers, which widen
    u32x4 kr[PASSES], vr[PASSES];
    uint32_t ksr[PASSES], vsr[PASSES];
    auto load_codes = [&](int seq, int kvh, int key0, const int (&e)[PASSES]) {
        size_t row[PASSES];
        rows_of(seq, kvh, key0, e, row);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            kr[i] = *(const u32x4*)((const uint8_t*)P.k + row[i] * D + lane * 16);
            vr[i] = *(const u32x4*)((const uint8_t*)P.v + row[i] * D + lane * 16);
            ksr[i] = (P.ks + row[i])[lrow];
            vsr[i] = (P.vs + row[i])[lrow];
        }
    };
    auto stage_codes = [&](int key0, int which, int lim0, int k1) {
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
    auto fetch = [&](int seq, int kvh, int key0, const int (&e)[PASSES], int which) {
        size_t row[PASSES];
        rows_of(seq, kvh, key0, e, row);
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
        const float m_use = (m_run == -INFINITY ? 0.f : m_run) - weight_shift<T>(8);       // (weights reach 2^8 times the maximum's)
        v8 pf[KS];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                pf[2 * b + (i >> 3)][i & 7] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s_acc[b][i], P.scale_log2e, -m_use));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) l_run = add_weights<T>(pf[ks], l_run);
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
        pages(I.seq, k0);
        if constexpr (Q8) { load_codes(I.seq, I.kvh, k0, pg); stage_codes(k0, 0, lim0, k1); }
        else fetch(I.seq, I.kvh, k0, pg, 0);
    }
    int cur = 0;
    for (bool first_unit = true;; first_unit = false) {
        // the next unit, looked up while this one's first tile is on its way: its own first one follows this one's last
        int nseq = I.seq, nkvh = I.kvh + 1, nsteps = steps;
        Rows nR = {I.first, I.rows, I.past, I.end};
        bool next = false;
        if constexpr (SHARED) {
            next = left > upto - from;
            if (next && nkvh == P.h_kv) {
                nkvh = 0;
                do { if (++nseq == P.n_seqs) break; nR = rows_of_seq<true>(P, nseq); nsteps = steps_of(nR.end); } while (nsteps == 0);
                next = nseq < P.n_seqs;
            }
            if (next) {
                const __attribute__((address_space(4))) int32_t* const t =
                    (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(P.map.table + (size_t)nseq * P.map.width);
#pragma unroll
                for (int i = 0; i < PASSES; ++i) {
                    const int at = (i * RPP + wave * RPW) >> P.map.shift;
                    npg[i] = t[at < P.map.width ? at : P.map.width - 1];
                }
            }
        }
        const int nleft = left - (upto - from);
        int nk1 = nleft < nsteps ? nleft * PAD_STEP : nR.end;
        nk1 = nk1 < nR.end ? nk1 : nR.end;
        m_run = -INFINITY; l_run = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i) o_acc[i] = floatx16{};
#pragma unroll
        for (int s = 0; s < QS; ++s) arrived(qf[s]);
        for (int key0 = k0; key0 < k1; key0 += PAT_BK, cur ^= 1) {
            if constexpr (!Q8) loads_done();
            __syncthreads();
            const int nxt = key0 + PAT_BK;
            const bool more = nxt < k1, over = SHARED && !more && next;
            if constexpr (Q8) {
                if (more) load_codes(I.seq, I.kvh, nxt, pg);
                else if (over) load_codes(nseq, nkvh, 0, npg);
            } else {
                if (key0 + PAT_BK - 1 > lim0) clean(key0, cur);
                if (more) fetch(I.seq, I.kvh, nxt, pg, cur ^ 1);
                else if (over) fetch(nseq, nkvh, 0, npg, cur ^ 1);
            }
            if (key0 <= lim_hi) compute(key0, cur, key0 + PAT_BK - 1 > lim_lo);
            if constexpr (Q8) {
                if (more) stage_codes(nxt, cur ^ 1, lim0, k1);
                else if (over) stage_codes(0, cur ^ 1, nR.past < nk1 ? nR.past : nk1 - 1, nk1);
            }
        }

        {
            unsigned a = __builtin_bit_cast(unsigned, l_run), c = a;
            lane_swap32(a, c);
            l_run = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, c);
        }
        const bool all = SHARED ? from == 0 && upto == steps : I.n_parts <= 1;
        if constexpr (SHARED) {
            if (from == 0 && tid == 0)              // where the join finds the unit's parts
                P.units[I.seq * P.h_kv + I.kvh] = int2{(int)(2 * blockIdx.x + (first_unit ? 0 : 1)), all ? 1 : 1 + (steps - upto + per - 1) / per};
        }
        if (live && all) {
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
        } else if (live) {
            const size_t pr = SHARED ? (size_t)(2 * blockIdx.x + (first_unit ? 0 : 1)) * P.tile_rows + r
                                     : ((size_t)I.split * P.n_rows + I.first + token) * P.n_heads + head;
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
        if (!next) return;
        left = nleft; from = 0; steps = nsteps;
        I.seq = nseq; I.kvh = nkvh; I.first = nR.first; I.past = nR.past; I.end = nR.end;
        I.rows = nR.rows < P.tile_rows ? nR.rows : P.tile_rows;
        at_unit();
        enter();
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
    const int first = P.cu_rows[seq], n = P.cu_rows[seq + 1] - first, past = past_of(P, P.seq_lens[seq]);
    if (first < 0 || t < first || n > P.n_rows - first) return;
    const int rows = n * P.group, r = (t - first) * P.group + head % P.group;
    if (r >= P.n_tiles * tile_rows) return;                 // rows that were left out
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

// Joins what the workgroups that share all units' keys left of a unit: NW waves a (row, head), each takes every NWth part, eight
// of them in flight at once.  A unit's first part lies where the workgroup that began it said, the others at the first place of
// the workgroups behind it.
template <typename T, int D, int NW>
__global__ void __launch_bounds__(256) paged_attention_join_rows_kernel(PagedAttnParams P) {
    constexpr int E = D / 64, MAX = 8;                      // outputs a lane, parts a wave at a time
    typedef float vecE __attribute__((ext_vector_type(E)));
    __shared__ float acc[4][D], sums[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * (4 / NW) + wave / NW;
    const int w = wave % NW, t = (int)(item / P.n_heads), head = (int)(item % P.n_heads);
    const int seq = t < P.n_rows ? __builtin_amdgcn_readfirstlane(seq_of_row(P.cu_rows, P.n_seqs, t)) : P.n_seqs;
    if (seq >= P.n_seqs) return;                            // (NW > 1: the whole block's row)
    const int first = P.cu_rows[seq], n = P.cu_rows[seq + 1] - first, r = (t - first) * P.group + head % P.group;
    if (first < 0 || n > P.n_rows - first || r < 0 || r >= P.tile_rows) return;       // rows that were left out
    const int2 u = P.units[seq * P.h_kv + head / P.group];
    // a unit without keys (a length below zero) has no parts, and nobody wrote its entry: its rows are zeros
    const bool none = attn_tile_end(P, past_of(P, P.seq_lens[seq]), n * P.group, 0, P.tile_rows) == 0;
    const int parts = __builtin_amdgcn_readfirstlane(none ? 0 : u.y), g0 = __builtin_amdgcn_readfirstlane(u.x);
    if (parts == 1) return;                                 // written already
    auto slot = [&](int p) { return (size_t)(p ? (g0 & ~1) + 2 * p : g0) * P.tile_rows + r; };
    float top = -INFINITY;
    for (int p = lane; p < parts; p += 64) top = fmaxf(top, P.part_ml[slot(p) * 2]);
    vecE mine = {};
    float sum = 0.f;
    for (int p0 = w; p0 < parts; p0 += NW * MAX) {
        vecE o[MAX];
        float m[MAX], l[MAX];
#pragma unroll
        for (int i = 0; i < MAX; ++i) {
            const size_t at = slot(p0 + NW * i < parts ? p0 + NW * i : p0);       // no branch: all of them are in flight
            m[i] = P.part_ml[at * 2];
            l[i] = P.part_ml[at * 2 + 1];
            o[i] = *(const vecE*)(P.part_o + at * D + lane * E);
        }
        if (p0 == w) top = wave_max_f32_dpp(top);
#pragma unroll
        for (int i = 0; i < MAX; ++i) {
            const float f = p0 + NW * i < parts && m[i] > -INFINITY ? __builtin_amdgcn_exp2f(m[i] - top) : 0.f;
            mine += o[i] * f;
            sum += l[i] * f;
        }
    }
    if constexpr (NW > 1) {
        *(vecE*)&acc[wave][lane * E] = mine;
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int i = 1; i < NW; ++i) { mine += *(const vecE*)&acc[i][lane * E]; sum += sums[i]; }
    }
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    T* dst = (T*)P.out + (size_t)t * P.out_stride + (size_t)head * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = (T)(mine[e] * inv);
}

struct AttnPlan { int tile_rows, n_tiles, n_splits, split_len, n_groups; size_t parts, bytes; };

static AttnPlan attn_plan(int n_seqs, int n_rows, int max_rows, int max_len, int n_heads, int h_kv, int d) {
    AttnPlan A = {};
    if (max_rows > n_rows) max_rows = n_rows;
    const int64_t rows = (int64_t)max_rows * (n_heads / h_kv), units = (int64_t)n_seqs * h_kv;
    A.n_tiles = A.n_splits = 1;
    A.split_len = max_len;
    // Shared evenly: few rows always; up to a tile of them where the units are neither few, whose keys the split below divides evenly
    // enough, nor as many as fit the card, which need no split.  Shared | split, six tokens of 64 / 8 heads over 300-4000 fp16 keys: 64
    // units 27.7 | 27.2 us, 128 39.5 | 45.3, 256 77 | 83, 384 of 2000 keys 99 | 118, 512 149 | 134, 768 175 | 154.
    if (rows <= 32 || (rows <= 128 && max_len > 256 && units >= 128 && units < 512)) {
        A.tile_rows = rows <= 16 ? 16 : (int)((rows + 31) / 32 * 32);
        // as many workgroups as fit the card (256 CUs; by registers and LDS), but none for fewer than 256 keys
        const int64_t fit = 256 * 2, most = units * ((max_len + 255) / 256);
        A.n_groups = max_len <= 256 ? 0 : (int)(fit < most ? fit : most);
        A.parts = (size_t)2 * A.n_groups * A.tile_rows;
        if (A.n_groups) A.bytes = A.parts * (d + 2) * sizeof(float) + units * sizeof(int2);
        return A;
    }
    A.tile_rows = 128;
    A.n_tiles = (int)((rows + 127) / 128);
    // Few tiles: the key axis is split for one round of the two workgroups that share a CU, in parts of 512 keys or more.  Parts are
    // dear here, 128 rows of fp32 sums each: with four rounds in parts of 256, 2048 rows of 32 heads took 157 us instead of 59.  Parts of
    // 256 keys where there are hardly any tiles: six tokens of 64 / 8 heads behind 1000 keys 12.7 instead of 17.0 us, behind 8000
    // 15.2 instead of 18.0; with 64 tiles 37.9 instead of 36.1; parts of 128 take longer from 8000 keys on (17.3).
    int64_t want = (512 + units * A.n_tiles - 1) / (units * A.n_tiles);
    want = want > 64 ? 64 : want;
    int64_t len = (max_len + want - 1) / want;
    const int64_t least = units * A.n_tiles <= 32 ? 256 : 512;
    len = len < least ? least : len;
    A.split_len = (int)((len + 127) / 128 * 128);
    A.n_splits = (max_len + A.split_len - 1) / A.split_len;
    if (A.n_splits > 1) A.bytes = (A.parts = (size_t)A.n_splits * n_rows * n_heads) * (d + 2) * sizeof(float);
    return A;
}

extern "C" size_t sq_paged_attention_workspace_bytes(int n_seqs, int n_rows, int max_rows, int max_len, int n_heads, int h_kv, int d) {
    if (n_seqs <= 0 || n_rows <= 0 || max_rows <= 0 || max_len <= 0 || n_heads <= 0 || h_kv <= 0 || n_heads % h_kv || d <= 0) return 0;
    return attn_plan(n_seqs, n_rows, max_rows, max_len, n_heads, h_kv, d).bytes;
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
    const AttnPlan A = attn_plan(n_seqs, n_rows, max_rows, max_len, n_heads, h_kv, d);
    if (A.bytes && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < A.bytes)) return SQ_EINVAL;
    const int64_t grid = A.n_groups ? A.n_groups : (int64_t)n_seqs * h_kv * A.n_tiles * A.n_splits, join = (int64_t)n_rows * n_heads;
    if (grid > PAGED_MAX_GRID || join > PAGED_MAX_GRID || (int64_t)n_seqs * h_kv * (max_len / 128 + 1) > 0x7fffffff) return SQ_EUNSUPPORTED;
    if (max_len > 1 << 30) return SQ_EUNSUPPORTED;          // keys are counted in 32 bits, some tiles past the end
    PagedAttnParams P = {q, q_head_stride, q_row_stride, k_pages, v_pages, (const uint8_t*)k_scales, (const uint8_t*)v_scales, out, out_stride,
                         {d_page_table, table_width, n_pages, shift}, d_seq_lens, d_cu_rows, n_seqs, n_rows, n_heads, h_kv, n_heads / h_kv,
                         scale * 1.4426950408889634f, max_len, A.n_tiles, A.n_splits, A.split_len, A.tile_rows, A.n_groups,
                         (float*)workspace, (float*)workspace + A.parts * d, (int2*)((float*)workspace + A.parts * (d + 2))};
    hipStream_t st = (hipStream_t)stream;
#define SQ_LAUNCH(K, G, ...) hipLaunchKernelGGL(K, dim3((unsigned)(G)), dim3(256), 0, st, __VA_ARGS__)
#define SQ_KERNELS(TT, DD, QQ) do { \
        if (A.tile_rows == 16) SQ_LAUNCH((paged_attention_rows_kernel<TT, DD, QQ, 1>), grid, P); \
        else if (A.tile_rows == 32) SQ_LAUNCH((paged_attention_rows_kernel<TT, DD, QQ, 2>), grid, P); \
        else if (A.n_groups) SQ_LAUNCH((paged_attention_tiles_kernel<TT, DD, QQ, true>), grid, P); \
        else SQ_LAUNCH((paged_attention_tiles_kernel<TT, DD, QQ, false>), grid, P); \
    } while (0)
    // the join of few rows gives each four waves (a part of the key axis each at a time), of many one
#define SQ_JOIN_ROWS(TT, DD) do { \
        if (join < 1024) SQ_LAUNCH((paged_attention_join_rows_kernel<TT, DD, 4>), join, P); \
        else SQ_LAUNCH((paged_attention_join_rows_kernel<TT, DD, 1>), (join + 3) / 4, P); \
    } while (0)
#define SQ_TYPES(TT, DD) do { \
        if (k_scales) SQ_KERNELS(TT, DD, true); else SQ_KERNELS(TT, DD, false); \
        if (A.n_groups) SQ_JOIN_ROWS(TT, DD); \
        else if (A.n_splits > 1) SQ_LAUNCH((paged_attention_join_kernel<TT, DD>), join, P, A.tile_rows); \
    } while (0)
    if (dtype == SQ_DTYPE_F16) { if (d == 128) SQ_TYPES(half_t, 128); else SQ_TYPES(half_t, 64); }
    else                       { if (d == 128) SQ_TYPES(bf16_t, 128); else SQ_TYPES(bf16_t, 64); }
#undef SQ_TYPES
#undef SQ_JOIN_ROWS
#undef SQ_KERNELS
#undef SQ_LAUNCH
    return sq_check_launch();
}
