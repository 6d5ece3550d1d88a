// Attention of new tokens over a paged cache: what its kernels share.
#pragma once
#include "cache_view.cuh"

namespace jsm {

struct ChunkArgs {
    CacheView c;
    const __nv_bfloat16* q;
    long long q_rs;
    __nv_bfloat16* out;
    long long out_rs;
    int T, max_new, max_context, Hq, G;  // G: query heads of a kv head
    int window;                          // 0: none
    float scale_log2;
};

// Sequences with a few new tokens only (chunk_few.cu).
struct FewPlan {
    int rows;    // of queries per kv head and group: 8 or 16
    int per;     // tokens of a group
    int tokens;  // of a sequence at most; the others are left to another kernel
    int n_runs;  // runs of pages
    bool merge;  // whether partial results can meet
    size_t bytes;
};
FewPlan chunk_few_plan(int n_seqs, int T, int max_new, int max_context, int Hkv, int G, int window, int rows, int tokens, int D, bool q8);
jsm_status chunk_few_launch(const ChunkArgs& a, const FewPlan& f, void* scratch, cudaStream_t st);

// sequences of more than few_tokens tokens
jsm_status chunk_flash_launch(const ChunkArgs& a, int few_tokens, cudaStream_t st);

#ifdef __CUDACC__
// lengths of a sequence that the kernels may rely on; false: no new tokens, or lengths that do not fit (an error)
template <bool EARLY = false>
__device__ __forceinline__ bool chunk_lengths(const ChunkArgs& a, int s, int& first_row, int& n_new, int& ctx) {
    if (!cache_lengths<EARLY>(a.c, s, a.T, first_row, n_new, ctx)) return false;
    if (n_new <= a.max_new && ctx <= a.max_context) return true;
    cache_error(a.c.err, CACHE_BAD_LENGTH);
    return false;
}
__device__ __forceinline__ int first_key(int window, int pos) { return window > 0 ? max(0, pos - window + 1) : 0; }

// One query row of one head by one warp, key after key in fp32, over exactly the keys that it sees: lane l has the components l * (D / 32) and up.
// sum of p v, sum of p, as p = 2^(score - largest so far); o is the quotient.  Values count 2^-32 of themselves until the end: a context has fewer than 2^31 keys, so a
// sum of the largest bf16 numbers stays one of fp32 (and what is below 2^-94 loses bits; a row that comes here for another reason has outputs exact to 2^-118).
template <int D, bool Q8>
__device__ __noinline__ void attend_row(const ChunkArgs& a, int s, int row, int head, int pos) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31, hk = head / a.G, last = pos;
    float q[N], o[N], m = -INFINITY, l = 0.0f;
    const __nv_bfloat16* src = a.q + row * a.q_rs + (long long)head * D + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = __bfloat162float(src[i]);
        o[i] = 0.0f;
    }
    int page = -1;
    for (int key = first_key(a.window, pos), at = -1; key <= last; ++key) {
        if (key / JSM_PAGE_SIZE != at) {
            at = key / JSM_PAGE_SIZE;
            page = cache_page(a.c, s, key);
        }
        if (page < 0) continue;
        float k[N], v[N], sum = 0.0f;
#pragma unroll
        for (int value = 0; value < 2; ++value) {
            const long long r = cache_row(a.c, page, value, hk, key);
            float(&x)[N] = value ? v : k;
            if constexpr (Q8) {
                const int8_t* p = static_cast<const int8_t*>(a.c.pool) + r * D + lane * N;
                const float scale = bf16_bits_to_f32(a.c.scales[r]);
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = __bfloat162float(__float2bfloat16_rn(__fmul_rn((float)p[i], scale)));
            } else {
                const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.c.pool) + r * D + lane * N;
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = __bfloat162float(p[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) sum = fmaf(q[i], k[i], sum);
        const float score = warp_sum(sum) * a.scale_log2;
        if (score == -INFINITY) {  // of weight 0 beside any other key, and 0 times an infinite value is no number
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = fmaf(0.0f, v[i], o[i]);
            continue;
        }
        const float mn = fmaxf(m, score), corr = exp2f(m - mn), p = exp2f(score - mn);
        m = mn;
        l = fmaf(l, corr, p);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(o[i], corr, p * (v[i] * 0x1p-32f));
    }
    __nv_bfloat16* dst = a.out + row * a.out_rs + (long long)head * D + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = __float2bfloat16_rn(o[i] / l * 0x1p32f);
}
#endif

}  // namespace jsm
