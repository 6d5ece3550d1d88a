// An 8-bit paged cache: new keys (rotated on the way) and values are quantised as they are written, and read back.
//
// A position's D components of one kv head share a scale:  a = max |x|,  s = a / 127 rounded up to bf16,  n = rint(x / s) (as x * (1 / s)), and the cache
// stands for bf16(n * s) - numbers of the type that the attention multiplies, so that every reader of the cache sees the same values, and one packed
// multiplication makes two of them.  The scale is rounded up so that |x| / s stays within 127.  a < 2^-100 gives s = 0; a NaN, an infinity or a > 2^127
// gives s = NaN: the whole row then reads back as NaN, which no reader can mistake for a number.
// Bound by memory: 4 D bytes in and 2 D + 4 bytes out per token and kv head.
#include "cache_view.cuh"
#include <math.h>

namespace jsm {

int* tc_error_word();

struct AppendArgs {
    CacheView c;
    const __nv_bfloat16 *k, *v;
    long long kv_rs;
    int T;
    const float2* table;  // rotation of the keys, or null
    int table_len, rot, adjacent;
};

constexpr float Q8_SMALLEST = 7.8886090522101180541e-31f;  // 2^-100
constexpr float Q8_LARGEST = 1.7014118346046923173e38f;    // 2^127: 127 s stays a bf16 number

// the scale of a row whose largest magnitude is `most`
__device__ __forceinline__ float q8_scale(float most) {
    if (most < Q8_SMALLEST) return 0.0f;
    if (!(most <= Q8_LARGEST)) return __uint_as_float(0x7FC00000u);
    return __uint_as_float((__float_as_uint(__fdiv_rn(most, 127.0f)) + 0xFFFFu) & 0xFFFF0000u);
}
__device__ __forceinline__ float q8_inverse(float scale) { return scale == 0.0f ? 0.0f : __fdiv_rn(1.0f, scale); }

// any pitches, alignments and rotations: one warp per (token, keys or values, kv head)
__global__ void __launch_bounds__(256) kv_append_q8_kernel(AppendArgs a) {
    __shared__ int found;
    chain_trigger();
    chain_wait();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.c.D;
    const int s = find_sequence(a.c, t, &found);
    if (s < 0) return;
    int first, n_new, ctx;
    if (!cache_lengths(a.c, s, a.T, first, n_new, ctx)) return;
    const int pos = ctx - n_new + t - first;
    if (a.table && pos >= a.table_len) {
        if (threadIdx.x == 0) cache_error(a.c.err, CACHE_BAD_POSITION);
        return;
    }
    const int page = cache_page(a.c, s, pos);
    if (page < 0) return;
    for (int r = warp; r < 2 * a.c.Hkv; r += 8) {
        const int value = r / a.c.Hkv, h = r % a.c.Hkv;
        const __nv_bfloat16* src = (value ? a.v : a.k) + t * a.kv_rs + (long long)h * D;
        float x[8], most = 0.0f;
        bool odd = false;  // (fmaxf passes over a NaN)
        for (int j = 0; j * 32 + lane < D; ++j) {
            const int i = j * 32 + lane;
            float y = __bfloat162float(src[i]);
            if (!value && a.table && i < a.rot) {
                const int half = a.rot / 2, pair = a.adjacent ? i / 2 : i % half;
                const bool second = a.adjacent ? i & 1 : i >= half;
                const int other = a.adjacent ? i ^ 1 : second ? i - half : i + half;
                const float2 e = a.table[(long long)pos * half + pair];
                const float z = __bfloat162float(src[other]);
                float y1, y2;
                rotate_pair(second ? z : y, second ? y : z, e.x, e.y, y1, y2);
                y = second ? y2 : y1;
            }
            x[j] = y;
            odd |= !(fabsf(y) <= 3.402823466e38f);
            most = fmaxf(most, fabsf(y));
        }
        most = warp_max(most);
        if (__any_sync(0xffffffffu, odd)) most = INFINITY;
        const float scale = q8_scale(most), inv = q8_inverse(scale);
        const long long row = cache_row(a.c, page, value, h, pos);
        int8_t* dst = static_cast<int8_t*>(a.c.pool) + row * D;
        for (int j = 0; j * 32 + lane < D; ++j) dst[j * 32 + lane] = (int8_t)__float2int_rn(__fmul_rn(x[j], inv));
        if (lane == 0) a.c.scales[row] = (uint16_t)(__float_as_uint(scale) >> 16);
    }
}

// Whole 16-byte pieces: LPR lanes have eight components each of a row (token, keys or values, kv head); a row's first loads do not wait for its page.  The partner of a
// half is fetched a second time (from L1) rather than passed between lanes: the lanes of a half are four to sixteen apart in four registers.
// Rounding to a whole number: adding 1.5 * 2^23 leaves it in the low bits of the sum.
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
    x[0] = bf16lo(w.x); x[1] = bf16hi(w.x); x[2] = bf16lo(w.y); x[3] = bf16hi(w.y);
    x[4] = bf16lo(w.z); x[5] = bf16hi(w.z); x[6] = bf16lo(w.w); x[7] = bf16hi(w.w);
}
template <int LPR>
__global__ void __launch_bounds__(256) kv_append_q8_vec_kernel(AppendArgs a) {
    constexpr int ROWS = 256 / LPR, U = 4;
    __shared__ int found;
    chain_trigger();
    chain_wait();
    const int t = blockIdx.x, D = a.c.D, Hkv = a.c.Hkv, n_rows = 2 * Hkv;
    const int i0 = threadIdx.x % LPR * 8, group = threadIdx.x / LPR;
    const bool on = i0 < D, turns = a.table && i0 < a.rot;
    const int half = a.rot / 2;
    const bool second = !a.adjacent && i0 >= half;
    uint4 w[U], w2[U];
    auto load = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * ROWS;
            if (r >= n_rows || !on) break;
            const __nv_bfloat16* src = (r < Hkv ? a.k + t * a.kv_rs + (long long)r * D : a.v + t * a.kv_rs + (long long)(r - Hkv) * D) + i0;
            w[u] = *reinterpret_cast<const uint4*>(src);
            if (r < Hkv && turns && !a.adjacent) w2[u] = *reinterpret_cast<const uint4*>(second ? src - half : src + half);
        }
    };
    load(group);
    const int s = find_sequence(a.c, t, &found);
    if (s < 0) return;
    int first, n_new, ctx;
    if (!cache_lengths(a.c, s, a.T, first, n_new, ctx)) return;
    const int pos = ctx - n_new + t - first;
    if (a.table && pos >= a.table_len) {
        if (threadIdx.x == 0) cache_error(a.c.err, CACHE_BAD_POSITION);
        return;
    }
    const int page = cache_page(a.c, s, pos);
    if (page < 0) return;
    float c[8], sn[8];  // adjacent: four pairs; halves: eight
    if (turns) {
        const float4* e = reinterpret_cast<const float4*>(a.table + (long long)pos * half + (a.adjacent ? i0 / 2 : second ? i0 - half : i0));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < 2 || !a.adjacent) {
                const float4 v = e[i];
                c[2 * i] = v.x; sn[2 * i] = v.y; c[2 * i + 1] = v.z; sn[2 * i + 1] = v.w;
            }
    }
    const int ahead = threadIdx.x % 32 / LPR;  // (a warp's rows take their turns together: lanes meet in shuffles)
    for (int r0 = group; r0 - ahead < n_rows; r0 += U * ROWS) {
        if (r0 != group) load(r0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * ROWS;
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, most = 0.0f, sum = 0.0f;
            if (r < n_rows && on) {
                unpack8(w[u], x);
                if (r < Hkv && turns) {
                    if (a.adjacent) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) rotate_pair(x[2 * i], x[2 * i + 1], c[i], sn[i], x[2 * i], x[2 * i + 1]);
                    } else {
                        float y[8];
                        unpack8(w2[u], y);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float y1, y2;
                            rotate_pair(second ? y[i] : x[i], second ? x[i] : y[i], c[i], sn[i], y1, y2);
                            x[i] = second ? y2 : y1;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    most = fmaxf(most, fabsf(x[i]));
                    sum += x[i] * 0.0f;  // a NaN where a component is one, or infinite (fmaxf passes over a NaN)
                }
                if (!(sum == 0.0f)) most = INFINITY;
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            if (r >= n_rows || !on) continue;
            const float scale = q8_scale(most), inv = q8_inverse(scale);
            uint32_t n[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.0f));
            uint2 o;
            o.x = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
            o.y = __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410);
            if (!(scale == scale)) o = make_uint2(0, 0);
            const long long row = r < Hkv ? cache_row(a.c, page, 0, r, pos) : cache_row(a.c, page, 1, r - Hkv, pos);
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(a.c.pool) + row * D + i0) = o;
            if (i0 == 0) a.c.scales[row] = (uint16_t)(__float_as_uint(scale) >> 16);
        }
    }
}

struct ReadArgs {
    CacheView c;
    void *k_out, *v_out;
    long long out_rs;
    int T, f32;
};

__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    __shared__ int found;
    chain_trigger();
    chain_wait();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.c.D;
    const int s = find_sequence(a.c, t, &found);
    if (s < 0) return;
    int first, n_new, ctx;
    if (!cache_lengths(a.c, s, a.T, first, n_new, ctx)) return;
    const int pos = ctx - n_new + t - first;
    const int page = cache_page(a.c, s, pos);
    if (page < 0) return;
    for (int r = warp; r < 2 * a.c.Hkv; r += 8) {
        const int value = r / a.c.Hkv, h = r % a.c.Hkv;
        const long long row = cache_row(a.c, page, value, h, pos), to = t * a.out_rs + (long long)h * D;
        const float scale = a.c.scales ? bf16_bits_to_f32(a.c.scales[row]) : 1.0f;
        for (int i = lane; i < D; i += 32) {
            const float x = a.c.scales ? (float)static_cast<const int8_t*>(a.c.pool)[row * D + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.c.pool)[row * D + i]);
            const __nv_bfloat16 y = a.c.scales ? __float2bfloat16_rn(__fmul_rn(x, scale)) : static_cast<const __nv_bfloat16*>(a.c.pool)[row * D + i];
            if (a.f32) static_cast<float*>(value ? a.v_out : a.k_out)[to + i] = __bfloat162float(y);
            else static_cast<__nv_bfloat16*>(value ? a.v_out : a.k_out)[to + i] = y;
        }
    }
}

// whole 16-byte pieces of the outputs: eight components per lane, four rows' loads in flight
template <int LPR, bool Q8, bool F32>
__global__ void __launch_bounds__(256) kv_read_vec_kernel(ReadArgs a) {
    constexpr int ROWS = 256 / LPR, U = 4;
    __shared__ int found;
    chain_trigger();
    chain_wait();
    const int t = blockIdx.x, D = a.c.D, Hkv = a.c.Hkv, n_rows = 2 * Hkv;
    const int i0 = threadIdx.x % LPR * 8, group = threadIdx.x / LPR;
    const int s = find_sequence(a.c, t, &found);
    if (s < 0 || i0 >= D) return;
    int first, n_new, ctx;
    if (!cache_lengths(a.c, s, a.T, first, n_new, ctx)) return;
    const int pos = ctx - n_new + t - first;
    const int page = cache_page(a.c, s, pos);
    if (page < 0) return;
    for (int r0 = group; r0 < n_rows; r0 += U * ROWS) {
        uint4 w[U];
        uint32_t scale[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * ROWS;
            if (r >= n_rows) break;
            const long long row = r < Hkv ? cache_row(a.c, page, 0, r, pos) : cache_row(a.c, page, 1, r - Hkv, pos);
            if constexpr (Q8) {
                const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.c.pool) + row * D + i0);
                w[u].x = v.x;
                w[u].z = v.y;
                scale[u] = a.c.scales[row] * 0x00010001u;
            } else {
                w[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.pool) + row * D + i0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * ROWS;
            if (r >= n_rows) break;
            uint4 o = w[u];
            if constexpr (Q8) {
                o.x = q8_value2(__byte_perm(w[u].x, 0, 0x1100), scale[u]);
                o.y = q8_value2(__byte_perm(w[u].x, 0, 0x3322), scale[u]);
                o.z = q8_value2(__byte_perm(w[u].z, 0, 0x1100), scale[u]);
                o.w = q8_value2(__byte_perm(w[u].z, 0, 0x3322), scale[u]);
            }
            const long long to = t * a.out_rs + (long long)(r < Hkv ? r : r - Hkv) * D + i0;
            void* out = r < Hkv ? a.k_out : a.v_out;
            if constexpr (F32) {
                float* dst = static_cast<float*>(out) + to;
                reinterpret_cast<float4*>(dst)[0] = make_float4(bf16lo(o.x), bf16hi(o.x), bf16lo(o.y), bf16hi(o.y));
                reinterpret_cast<float4*>(dst)[1] = make_float4(bf16lo(o.z), bf16hi(o.z), bf16lo(o.w), bf16hi(o.w));
            } else {
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to) = o;
            }
        }
    }
}
template <int LPR>
static cudaError_t read_vec_launch(const ReadArgs& a, cudaStream_t st) {
    if (a.c.scales) return a.f32 ? launch_chained(kv_read_vec_kernel<LPR, true, true>, dim3(a.T), dim3(256), 0, st, a) : launch_chained(kv_read_vec_kernel<LPR, true, false>, dim3(a.T), dim3(256), 0, st, a);
    return a.f32 ? launch_chained(kv_read_vec_kernel<LPR, false, true>, dim3(a.T), dim3(256), 0, st, a) : launch_chained(kv_read_vec_kernel<LPR, false, false>, dim3(a.T), dim3(256), 0, st, a);
}

// what the calls over a paged cache check alike
jsm_status cache_view_check(const char* who, CacheView& c, void* pool, void* scales, int n_pages, const int32_t* table, int max_pages, const int32_t* starts,
                            const int32_t* context_lens, int n_seqs, int T, int Hkv, int D) {
    if (n_seqs < 0 || T < 0) JSM_FAIL(JSM_INVALID_ARG, "%s: %d sequences, %d rows", who, n_seqs, T);
    if (Hkv <= 0 || D <= 0 || D % 16 || D > 256) JSM_FAIL(JSM_SHAPE, "%s: %d kv heads of %d (a multiple of 16, up to 256)", who, Hkv, D);
    if (n_pages <= 0 || max_pages <= 0) JSM_FAIL(JSM_INVALID_ARG, "%s: a pool of %d pages, a table of %d", who, n_pages, max_pages);
    if (max_pages > INT32_MAX / JSM_PAGE_SIZE) JSM_FAIL(JSM_UNSUPPORTED, "%s: %d pages of a sequence", who, max_pages);
    if ((int64_t)n_pages * Hkv > INT32_MAX / (2 * JSM_PAGE_SIZE)) JSM_FAIL(JSM_UNSUPPORTED, "%s: %d pages of %d kv heads (2^31 rows of a head and more)", who, n_pages, Hkv);
    c = CacheView{pool, static_cast<uint16_t*>(scales), n_pages, table, max_pages, starts, context_lens, n_seqs, Hkv, D, nullptr};
    if (T == 0 || n_seqs == 0) return JSM_OK;
    if (!pool || !table || !starts || !context_lens) JSM_FAIL(JSM_INVALID_ARG, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(pool) & 15) || (reinterpret_cast<uintptr_t>(scales) & 15)) JSM_FAIL(JSM_INVALID_ARG, "%s: the pool must be 16-byte aligned", who);
    c.err = tc_error_word();
    return JSM_OK;
}

}  // namespace jsm

using namespace jsm;

extern "C" jsm_status jsm_kv_append_q8(void* d_pool, void* d_scales, int n_pages, const int32_t* d_block_table, int max_pages, const void* d_k, const void* d_v,
                                       int64_t kv_row_stride, const int32_t* d_starts, const int32_t* d_context_lens, int n_seqs, int T, int Hkv, int D,
                                       const float* d_rope_table, int table_len, int rot_dim, int layout, void* stream) {
    AppendArgs a{};
    const jsm_status s = cache_view_check("jsm_kv_append_q8", a.c, d_pool, d_scales, n_pages, d_block_table, max_pages, d_starts, d_context_lens, n_seqs, T, Hkv, D);
    if (s != JSM_OK) return s;
    if (d_rope_table) {
        if (rot_dim <= 0 || rot_dim % 2 || rot_dim > D) JSM_FAIL(JSM_SHAPE, "jsm_kv_append_q8: rotation of %d components of a head of %d", rot_dim, D);
        if (layout != JSM_ROPE_ADJACENT && layout != JSM_ROPE_HALF) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_append_q8: layout %d", layout);
        if (table_len <= 0 || (reinterpret_cast<uintptr_t>(d_rope_table) & 7)) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_append_q8: a table of %d positions, 8-byte aligned", table_len);
    }
    if (T == 0 || n_seqs == 0) return JSM_OK;
    if (!d_scales || !d_k || !d_v) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_append_q8: null pointer");
    if (kv_row_stride < (int64_t)Hkv * D) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_append_q8: rows of %lld elements for %d heads of %d", (long long)kv_row_stride, Hkv, D);
    if ((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 1) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_append_q8: rows that are not aligned to their elements");
    a.k = static_cast<const __nv_bfloat16*>(d_k);
    a.v = static_cast<const __nv_bfloat16*>(d_v);
    a.kv_rs = kv_row_stride;
    a.T = T;
    a.table = reinterpret_cast<const float2*>(d_rope_table);
    a.table_len = table_len; a.rot = rot_dim; a.adjacent = layout == JSM_ROPE_ADJACENT;
    const uintptr_t at = reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v) | reinterpret_cast<uintptr_t>(d_rope_table);
    const bool pieces = !(at & 15) && kv_row_stride % 8 == 0 && (!d_rope_table || (layout == JSM_ROPE_ADJACENT ? rot_dim : rot_dim / 2) % 8 == 0);
    JSM_CUDA_CHECK(!pieces    ? launch_chained(kv_append_q8_kernel, dim3(T), dim3(256), 0, as_stream(stream), a)
                   : D <= 64  ? launch_chained(kv_append_q8_vec_kernel<8>, dim3(T), dim3(256), 0, as_stream(stream), a)
                   : D <= 128 ? launch_chained(kv_append_q8_vec_kernel<16>, dim3(T), dim3(256), 0, as_stream(stream), a)
                              : launch_chained(kv_append_q8_vec_kernel<32>, dim3(T), dim3(256), 0, as_stream(stream), a));
    JSM_LAUNCH_CHECK();
    return JSM_OK;
}

extern "C" jsm_status jsm_kv_read(const void* d_pool, const void* d_scales, int n_pages, const int32_t* d_block_table, int max_pages, const int32_t* d_starts,
                                  const int32_t* d_context_lens, int n_seqs, int T, int Hkv, int D, void* d_k_out, void* d_v_out, int64_t out_row_stride,
                                  jsm_dtype out_dtype, void* stream) {
    ReadArgs a{};
    const jsm_status s = cache_view_check("jsm_kv_read", a.c, const_cast<void*>(d_pool), const_cast<void*>(d_scales), n_pages, d_block_table, max_pages, d_starts,
                                          d_context_lens, n_seqs, T, Hkv, D);
    if (s != JSM_OK) return s;
    if (out_dtype != JSM_F32 && out_dtype != JSM_BF16) JSM_FAIL(JSM_UNSUPPORTED, "jsm_kv_read: dtype %d", (int)out_dtype);
    if (T == 0 || n_seqs == 0) return JSM_OK;
    if (!d_k_out || !d_v_out) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_read: null pointer");
    if (out_row_stride < (int64_t)Hkv * D) JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_read: rows of %lld elements for %d heads of %d", (long long)out_row_stride, Hkv, D);
    if ((reinterpret_cast<uintptr_t>(d_k_out) | reinterpret_cast<uintptr_t>(d_v_out)) & (out_dtype == JSM_F32 ? 3 : 1))
        JSM_FAIL(JSM_INVALID_ARG, "jsm_kv_read: rows that are not aligned to their elements");
    a.k_out = d_k_out; a.v_out = d_v_out; a.out_rs = out_row_stride; a.T = T; a.f32 = out_dtype == JSM_F32;
    const bool pieces = !((reinterpret_cast<uintptr_t>(d_k_out) | reinterpret_cast<uintptr_t>(d_v_out)) & 15) && out_row_stride % (a.f32 ? 4 : 8) == 0;
    JSM_CUDA_CHECK(!pieces    ? launch_chained(kv_read_kernel, dim3(T), dim3(256), 0, as_stream(stream), a)
                   : D <= 64  ? read_vec_launch<8>(a, as_stream(stream))
                   : D <= 128 ? read_vec_launch<16>(a, as_stream(stream))
                              : read_vec_launch<32>(a, as_stream(stream)));
    JSM_LAUNCH_CHECK();
    return JSM_OK;
}
