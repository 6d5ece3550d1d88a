// What the operators over sequences of a paged cache share: which sequence a row of new tokens belongs to, where a position lies in the pool, and
// how a sequence's lengths are checked on the device.
//
// Row t of the new tokens belongs to the sequence s with starts[s] <= t < starts[s + 1]; context_lens[s] counts the new tokens, so row t is
// position context_lens[s] - (starts[s + 1] - t).  Pool: [page][keys, values][kv head][64 positions][D], bf16 or int8; an int8 pool has a bf16
// scale per position, [page][keys, values][kv head][64], and stands for bf16(number * scale).
#pragma once
#include "common.cuh"

namespace jsm {

// codes of the device error word (jsm_check_device_errors)
enum CacheError : int { CACHE_BAD_POSITION = 33, CACHE_BAD_PAGE = 34, CACHE_BAD_LENGTH = 35 };

struct CacheView {
    void* pool;
    uint16_t* scales;            // null: a bf16 pool
    int n_pages;
    const int32_t* table;        // [n_seqs][max_pages]
    int max_pages;
    const int32_t* starts;       // [n_seqs + 1]
    const int32_t* context_lens; // [n_seqs]
    int n_seqs, Hkv, D;
    int* err;
};

#ifdef __CUDACC__
__device__ __forceinline__ void cache_error(int* err, int code) {
    if (err) atomicCAS(err, 0, code);
}

// of a sequence whose first row is not its end: ascending, rows of the call, a context that holds them and that the table's row holds
__device__ __forceinline__ bool lengths_fit(const CacheView& c, int T, int first_row, int end, int ctx) {
    if (first_row >= 0 && end > first_row && end <= T && ctx >= end - first_row && (ctx - 1) / JSM_PAGE_SIZE < c.max_pages) return true;
    cache_error(c.err, CACHE_BAD_LENGTH);
    return false;
}
// new tokens and context of sequence s; false (and an error) where they do not fit the table or one another.  EARLY: for a kernel that has not waited for its predecessor (past L1)
template <bool EARLY = false>
__device__ __forceinline__ bool cache_lengths(const CacheView& c, int s, int T, int& first_row, int& n_new, int& ctx) {
    auto load = [](const int32_t* p) { return EARLY ? load_early(p) : *p; };
    first_row = load(c.starts + s);
    const int end = load(c.starts + s + 1);
    n_new = end - first_row;
    ctx = load(c.context_lens + s);
    return end != first_row && lengths_fit(c, T, first_row, end, ctx);
}

// The sequence of row t of the T rows, for a whole block: every thread looks at one sequence, one round of loads for as many sequences as the block has threads.  -1: none.
// Sequences that no row leads to because their own rows do not fit are reported here.
__device__ __forceinline__ int find_sequence(const CacheView& c, int t, int T, int* found) {
    if (threadIdx.x == 0) *found = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < c.n_seqs; s += blockDim.x) {
        const int from = c.starts[s], to = c.starts[s + 1];
        if (from <= t && t < to) *found = s;
        if (from != to && (from < 0 || to < from || to > T)) cache_error(c.err, CACHE_BAD_LENGTH);
    }
    __syncthreads();
    return *found;
}

// page of a position of sequence s (within its table row); -1 and an error for an entry outside the pool
__device__ __forceinline__ int cache_page(const CacheView& c, int s, int pos) {
    const int page = c.table[(long long)s * c.max_pages + pos / JSM_PAGE_SIZE];
    if (page >= 0 && page < c.n_pages) return page;
    cache_error(c.err, CACHE_BAD_PAGE);
    return -1;
}
// row of a position (elements / D of the pool, and the index of its scale); value: 0 keys, 1 values
__device__ __forceinline__ long long cache_row(const CacheView& c, int page, int value, int head, int pos) {
    return (((long long)page * 2 + value) * c.Hkv + head) * JSM_PAGE_SIZE + pos % JSM_PAGE_SIZE;
}

// shared memory by its 32-bit address: a pointer that has been rounded up is generic to the compiler, with 64-bit arithmetic for every access
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Two numbers of an 8-bit cache, in the low bytes of the halves of p, times their scales: the values that the cache stands for.  0x4300 | the low seven bits is 128 + them
// as bf16, 0x4300 | the sign bit is 128 or 256; the difference is the number, exactly, and its product with the scale is rounded once.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t q8_value2(uint32_t p, uint32_t scale2) {
    const uint32_t lo = and_or(p, 0x007F007Fu, 0x43004300u), hi = and_or(p, 0x00800080u, 0x43004300u);
    uint32_t n, r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(n) : "r"(lo), "r"(hi));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(n), "r"(scale2));
    return r;
}

// rotation of a pair, every product rounded on its own
__device__ __forceinline__ void rotate_pair(float x1, float x2, float c, float s, float& y1, float& y2) {
    y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
}
#endif

}  // namespace jsm
