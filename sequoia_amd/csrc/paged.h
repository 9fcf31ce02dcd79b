// Shared by the paged-cache kernels (paged_kv.hip, paged_attention.hip): element types, page geometry, e4m3 rows.
//
// A layer's pages are [n_pages][H_kv][P][D], P a power of two from 16 to 256: a page of a KV head is the same [rows][D] block as
// the static slab, so a 16-row tile of keys never straddles two pages.  Row j of sequence b lives in page
// table[b][j >> shift], row j & (P - 1).
//
// An e4m3 row keeps one exponent byte x: value = code * 2^(x - 127).  The scale is a power of two so that what is lost is the ONE
// rounding to e4m3's four significant bits (at most 2^-4 relative, 2^(x - 137) absolute below the format's normal range): dividing by
// it never rounds, and multiplying by it only where the element type ends -- the smallest codes of fp16 rows of at most 448 * 2^-16
// (0.007), whose steps lie under fp16's own of 2^-24, and of bf16 rows of 2^-116; values above the type's largest are infinities,
// which the writer leaves none of.  Every reader of a type gets the same value.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct vec_of;
template <> struct vec_of<half_t> { typedef half8 v8; typedef half4 v4; typedef half2v v2; };
template <> struct vec_of<bf16_t> { typedef bf8v v8; typedef bf4v v4; typedef bf2v v2; };

struct PageMap {
    const int32_t* table;       // [n_seqs][width]
    int width, n_pages, shift;  // P = 1 << shift
};

// page of block `i` of sequence `b`, or -1 where the table holds none: an entry outside the pool is never followed
__device__ __forceinline__ int page_of(const PageMap& M, int b, int i) {
    if ((unsigned)i >= (unsigned)M.width) return -1;
    const int p = M.table[(size_t)b * M.width + i];
    return (unsigned)p < (unsigned)M.n_pages ? p : -1;
}

// Workgroups of up to 256 threads that one launch takes: the threads of a grid dimension are counted in 32 bits
#define PAGED_MAX_GRID 0xffffff

static inline int page_shift(int page_size) {
    for (int s = 4; s <= 8; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

// A table entry by wave-uniform index, loaded without a branch and looked at only where it is used (check_page), so that the wait
// for it falls behind the loads issued after it; one that is no page of the pool (only behind a table that ends early) becomes
// page 0, in bounds.
__device__ __forceinline__ int page_entry(const PageMap& M, int seq, int i) {
    i = i < M.width - 1 ? i : M.width - 1;
    return M.table[(size_t)seq * M.width + (i > 0 ? i : 0)];
}
__device__ __forceinline__ int check_page(const PageMap& M, int entry) {
    const int p = __builtin_amdgcn_readfirstlane(entry);
    return (unsigned)p < (unsigned)M.n_pages ? p : 0;
}

// The sequence that row `t` of a ragged batch belongs to (n_seqs: none), by one wave: the first that ends behind t.  64 ends a load
// instead of a search's chain of dependent ones.
__device__ __forceinline__ int seq_of_row(const int32_t* cu_rows, int n_seqs, int t) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < n_seqs; base += 64) {
        const uint64_t hit = __ballot(base + lane < n_seqs && cu_rows[base + lane + 1] > t);
        if (hit) return base + __builtin_ctzll(hit);
    }
    return n_seqs;
}

// 16 codes -> 16 values of T, rounded only where T ends: v_cvt_scalef32 multiplies by the power of two while it widens
template <typename T>
__device__ __forceinline__ void e4m3_expand(u32x4 codes, float scale, typename vec_of<T>::v8& lo, typename vec_of<T>::v8& hi) {
    typename vec_of<T>::v2 p[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (__is_same(T, half_t)) {
            p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], scale, false);
            p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], scale, true);
        } else {
            p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], scale, false);
            p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], scale, true);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[2 * i] = p[i][0]; lo[2 * i + 1] = p[i][1];
        hi[2 * i] = p[4 + i][0]; hi[2 * i + 1] = p[4 + i][1];
    }
}
// exponent byte -> scale; the writer's bytes lie in [1, 254]
__device__ __forceinline__ float e4m3_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
