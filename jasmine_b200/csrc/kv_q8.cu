// An 8-bit paged cache: new keys (rotated on the way) and values are quantised as they are written, and read back.
//
// A position's D components of one kv head share a scale:  a = max |x|,  s = a / 127 rounded up to bf16,  n = rint(x / s) (as x * (1 / s)), and the cache
// stands for bf16(n * s) - numbers of the type that the attention multiplies, so that every reader of the cache sees the same values, and one packed
// multiplication makes two of them.  The scale is rounded up so that |x| / s stays within 127.  a < 2^-100 gives s = 0; a NaN, an infinity or a > 2^127
// gives s = NaN: the whole row then reads back as NaN, which no reader can mistake for a number.
// Bound by memory: 4 D bytes in and 2 D + 4 bytes out per token and kv head.
#include "cache_view.cuh"
#include <limits.h>
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

// The scale of a row whose largest magnitude is `most` (NaN: the row has one).  The quotient by 127 is correctly rounded: Markstein's theorem ("Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990) for the correctly rounded reciprocal of the divisor, one residual and one correction.
__device__ __forceinline__ float q8_scale(float most) {
    constexpr float INV = 1.0f / 127.0f;
    const float q = __fmul_rn(most, INV), s = __fmaf_rn(__fmaf_rn(-127.0f, q, most), INV, q);
    if (most < Q8_SMALLEST) return 0.0f;
    return most <= Q8_LARGEST ? __uint_as_float((__float_as_uint(s) + 0xFFFFu) & 0xFFFF0000u) : __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ float q8_inverse(float scale) { return scale == 0.0f ? 0.0f : __frcp_rn(scale); }
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays one
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// any pitches and alignments: one warp per (token, keys or values, kv head)
__global__ void __launch_bounds__(256) kv_append_q8_kernel(AppendArgs a) {
    __shared__ int found;
    chain_trigger();
    chain_wait();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.c.D;
    const int s = find_sequence(a.c, t, a.T, &found);
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
            most = max_nan(most, fabsf(y));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float scale = q8_scale(most), inv = q8_inverse(scale);
        const long long row = cache_row(a.c, page, value, h, pos);
        int8_t* dst = static_cast<int8_t*>(a.c.pool) + row * D;
        for (int j = 0; j * 32 + lane < D; ++j) dst[j * 32 + lane] = (int8_t)__float2int_rn(__fmul_rn(x[j], inv));
        if (lane == 0) a.c.scales[row] = (uint16_t)(__float_as_uint(scale) >> 16);
    }
}

// The places of up to PLACES consecutive rows of new tokens from t0 on, for a whole block: position, and row of the pool of kv head 0's key (-1: the row is left alone); row r of the
// token's keys and values, keys of all heads first, lies JSM_PAGE_SIZE * r behind it
constexpr int PLACES = 16;
template <typename F>
__device__ __forceinline__ void find_places(const CacheView& c, int T, int t0, int n, int table_len, int* seq, int* pos, int* base, F beside) {
    if (threadIdx.x < PLACES) seq[threadIdx.x] = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < c.n_seqs; s += blockDim.x) {
        const int from = c.starts[s], to = c.starts[s + 1], ctx = c.context_lens[s];  // (one round of loads; the table is the other)
        const int k0 = max(0, from - t0), k1 = to > t0 ? min(n, to - t0) : 0;
        if (from != to && lengths_fit(c, T, from, to, ctx))
            for (int k = k0; k < k1; ++k) {
                seq[k] = s;
                pos[k] = ctx - to + t0 + k;
            }
    }
    __syncthreads();
    beside();  // (positions are known, pages not yet)
    if (threadIdx.x < n) {
        const int k = threadIdx.x, s = seq[k];
        int p = -1;
        if (s >= 0) {
            if (pos[k] < table_len) p = cache_page(c, s, pos[k]);
            else cache_error(c.err, CACHE_BAD_POSITION);
        }
        base[k] = p < 0 ? -1 : (int)cache_row(c, p, 0, 0, pos[k]);
    }
    __syncthreads();
}

// Whole 16-byte pieces: LPR lanes have two pieces of eight components each of a row (token, keys or values, kv head), up to PLACES tokens per block; a thread's first loads do not
// wait for the places.  A lane's pieces hold both components of its pairs (halves: a piece of each half), so that a rotation stays within the lane.
// Products that are rounded on their own before a sum: two by one instruction, the sums one by one (mul2).  Rounding to a whole number:
// adding 1.5 * 2^23 leaves it in the low bits of the sum.
// Prompts of 7887 tokens of 32 kv heads of 128 (194 MB in and out) 38 us alone, 5.1 TB/s of the measured 6.5 (44 between read-backs): latency at five blocks per multiprocessor.  A token's table entries are in shared
// memory: in registers they cost a block per multiprocessor, and a fetch in the middle of the rows (47 us).  The loads of two turns at a time, none while they are worked out, addresses in 64
// bits: 53 us; a lane per eight components with the partner of a half fetched a second time 74 us.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {  // of the magnitudes; a NaN stays one
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two products, each rounded (sums of them one by one: with add.rn.f32x2 behind mul.rn.f32x2 the results of 1024 random triples had the bits of one rounding, with scalar sums those of two)
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b, float c, float d) {
    asm("{ .reg .b64 p, q; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %5}; mul.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p; }" : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}
// row r of token k, and the one `step` rows on
__device__ __forceinline__ void advance(int& k, int& r, int step, int per_token) {
    r += step;
    if (r >= per_token) {
        r -= per_token;
        ++k;
        if (r >= per_token) {
            k += r / per_token;
            r %= per_token;
        }
    }
}
enum { TURN_NONE = 0, TURN_ADJACENT = 1, TURN_HALF = 2, TURN_ANY = 3 };  // any: parts that are no multiple of 16, element by element
template <int LPR, int TURN>
__global__ void __launch_bounds__(256, TURN == TURN_ANY ? 4 : 5) kv_append_q8_vec_kernel(AppendArgs a, int per_block) {
    constexpr int ROWS = 256 / LPR;  // rows of a block's turn
    __shared__ int sh_seq[PLACES], sh_pos[PLACES], sh_base[PLACES];
    __shared__ float4 sh_turn[TURN == TURN_ADJACENT || TURN == TURN_HALF ? PLACES * LPR * 4 : 1];  // of each token: two entries in 16 bytes, four of them for a lane, exchanged by lane
    chain_trigger();
    chain_wait();
    const int D = a.c.D, Hkv = a.c.Hkv, per_token = 2 * Hkv, t0 = blockIdx.x * per_block, n_tokens = min(per_block, a.T - t0), n_rows = n_tokens * per_token;
    const int l = threadIdx.x % LPR, group = threadIdx.x / LPR, half = a.rot / 2;
    const bool on = l * 16 < D, turns = TURN != TURN_NONE && l * 16 < a.rot;
    const int i0 = TURN == TURN_HALF && turns ? l * 8 : l * 16, i1 = TURN == TURN_HALF && turns ? i0 + half : i0 + 8;  // first components of the lane's pieces
    // rows of the block, token after token, keys before values: row r of token k (a block's rows lie within 2^31 elements)
    const int pitch = (int)a.kv_rs, apart = i1 - i0;
    const __nv_bfloat16 *k_src = a.k + t0 * a.kv_rs + i0, *v_src = a.v + t0 * a.kv_rs + i0 - (long long)Hkv * D;
    uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    auto load = [&](int k, int r) {
        if (!on || k >= n_tokens) return;
        const __nv_bfloat16* src = (r < Hkv ? k_src : v_src) + (k * pitch + r * D);
        w[0] = *reinterpret_cast<const uint4*>(src);
        w[1] = *reinterpret_cast<const uint4*>(src + apart);
    };
    int k = 0, r = 0;
    advance(k, r, group, per_token);
    load(k, r);
    const int ahead = threadIdx.x % 32 / LPR;  // (a warp's rows take their turns together: lanes meet in shuffles)
    find_places(a.c, a.T, t0, n_tokens, TURN != TURN_NONE ? a.table_len : INT_MAX, sh_seq, sh_pos, sh_base, [&] {
        if constexpr (TURN == TURN_ADJACENT || TURN == TURN_HALF) {
            const int pieces = half / 2;  // of a token's entries
            for (int i = threadIdx.x; i < n_tokens * pieces; i += 256) {
                const int token = i / pieces, c = i - token * pieces;
                if (sh_seq[token] >= 0 && sh_pos[token] < a.table_len)
                    sh_turn[token * (LPR * 4) + (c ^ ((c >> 3) & 3))] = reinterpret_cast<const float4*>(a.table + (long long)sh_pos[token] * half)[c];
            }
        }
    });
    for (int row = group; row - ahead < n_rows; row += ROWS) {
        const int base = k < n_tokens ? sh_base[k] : -1;
        float x[16];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const uint32_t in[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[p * 8 + 2 * i] = bf16lo(in[i]);
                x[p * 8 + 2 * i + 1] = bf16hi(in[i]);
            }
        }
        const int k_now = k, r_now = r;
        advance(k, r, ROWS, per_token);
        load(k, r);  // (the next turn's, while this one is worked out)
        if (TURN == TURN_ANY && r_now < Hkv && turns && base >= 0) {
            const __nv_bfloat16* src = a.k + (t0 + k_now) * a.kv_rs + r_now * D;
            const float2* e = a.table + (long long)sh_pos[k_now] * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int d = l * 16 + i;
                if (d >= a.rot) break;
                const bool second = a.adjacent ? d & 1 : d >= half;
                const float2 v = e[a.adjacent ? d / 2 : second ? d - half : d];
                const float z = __bfloat162float(src[a.adjacent ? d ^ 1 : second ? d - half : d + half]);
                x[i] = __fadd_rn(__fmul_rn(x[i], v.x), __fmul_rn(z, second ? v.y : -v.y));
            }
        } else if (TURN != TURN_NONE && TURN != TURN_ANY && r_now < Hkv) {
            if (turns) {  // (of a token without a place anything: it is not stored)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int c = l * 4 + i / 2;
                    const float4 e = sh_turn[min(k_now, PLACES - 1) * (LPR * 4) + (c ^ ((c >> 3) & 3))];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int i1_ = TURN == TURN_ADJACENT ? 2 * (i + h) : i + h, i2_ = TURN == TURN_ADJACENT ? 2 * (i + h) + 1 : i + h + 8;
                        rotate_pair(x[i1_], x[i2_], h ? e.z : e.x, h ? e.w : e.y, x[i1_], x[i2_]);
                    }
                }
            }
        }
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) most = max3_abs(most, x[i], x[i + 1]);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float scale = q8_scale(most), inv = q8_inverse(scale);
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            uint32_t n[4];  // 1.5 * 2^23 + the number
            float y[4];
            mul2(y[0], y[1], x[i], x[i + 1], inv, inv);
            mul2(y[2], y[3], x[i + 2], x[i + 3], inv, inv);
#pragma unroll
            for (int j = 0; j < 4; ++j) n[j] = __float_as_uint(__fadd_rn(y[j], 12582912.0f));
            out[i / 4] = scale == scale ? __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410) : 0u;
        }
        if (on && base >= 0) {
            const int to = base + r_now * JSM_PAGE_SIZE;
            int8_t* dst = static_cast<int8_t*>(a.c.pool) + (long long)to * D;
            if (TURN == TURN_HALF) {
                *reinterpret_cast<uint2*>(dst + i0) = make_uint2(out[0], out[1]);
                *reinterpret_cast<uint2*>(dst + i1) = make_uint2(out[2], out[3]);
            } else {
                *reinterpret_cast<uint4*>(dst + i0) = make_uint4(out[0], out[1], out[2], out[3]);
            }
            if (l == 0) a.c.scales[to] = (uint16_t)(__float_as_uint(scale) >> 16);
        }
    }
}
template <int LPR>
static cudaError_t append_vec_launch(const AppendArgs& a, int per_block, cudaStream_t st) {
    const dim3 grid((a.T + per_block - 1) / per_block);
    if (!a.table) return launch_chained(kv_append_q8_vec_kernel<LPR, TURN_NONE>, grid, dim3(256), 0, st, a, per_block);
    if (a.rot % 16 || (reinterpret_cast<uintptr_t>(a.table) & 15)) return launch_chained(kv_append_q8_vec_kernel<LPR, TURN_ANY>, grid, dim3(256), 0, st, a, per_block);
    return a.adjacent ? launch_chained(kv_append_q8_vec_kernel<LPR, TURN_ADJACENT>, grid, dim3(256), 0, st, a, per_block)
                      : launch_chained(kv_append_q8_vec_kernel<LPR, TURN_HALF>, grid, dim3(256), 0, st, a, per_block);
}

// Tokens of a block: what finding their places costs is worth eight rows of every thread (a block per token: 4 % slower for 32 kv heads, 27 % for 8), but the chip has eight blocks per
// multiprocessor first.
static int tokens_per_block(int T, int Hkv, int lanes) {
    const int rows = 8 * (256 / lanes) / (2 * Hkv), blocks = T / (8 * sm_count()), n = rows < blocks ? rows : blocks;
    return n < 1 ? 1 : n < PLACES ? n : PLACES;
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
    const int s = find_sequence(a.c, t, a.T, &found);
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

// whole 16-byte pieces of the outputs: eight components per lane, four rows' loads in flight, up to PLACES tokens per block.  The same prompts read back: 42 us alone, 4.6 TB/s (37 behind
// the append, from L2 in part); to fp32 85 us, 3.8 TB/s; a bf16 cache to bf16 43 us, 6.0 TB/s, to fp32 79 us, 4.9 TB/s.
template <int LPR, bool Q8, bool F32>
__global__ void __launch_bounds__(256) kv_read_vec_kernel(ReadArgs a, int per_block) {
    constexpr int ROWS = 256 / LPR, U = 4;
    __shared__ int sh_seq[PLACES], sh_pos[PLACES], sh_base[PLACES];
    chain_trigger();
    chain_wait();
    const int D = a.c.D, Hkv = a.c.Hkv, per_token = 2 * Hkv, t0 = blockIdx.x * per_block, n_tokens = min(per_block, a.T - t0);
    const int i0 = threadIdx.x % LPR * 8, group = threadIdx.x / LPR;
    find_places(a.c, a.T, t0, n_tokens, INT_MAX, sh_seq, sh_pos, sh_base, [] {});
    if (i0 >= D) return;
    int k = 0, r = 0;
    advance(k, r, group, per_token);
    while (k < n_tokens) {
        uint4 w[U];
        uint32_t scale[U];
        int k1 = k, r1 = r;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k1 >= n_tokens) break;
            if (sh_base[k1] >= 0) {
                const int at = sh_base[k1] + r1 * JSM_PAGE_SIZE;
                if constexpr (Q8) {
                    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.c.pool) + (long long)at * D + i0);
                    w[u].x = v.x;
                    w[u].z = v.y;
                    scale[u] = a.c.scales[at] * 0x00010001u;
                } else {
                    w[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.pool) + (long long)at * D + i0);
                }
            }
            advance(k1, r1, ROWS, per_token);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k >= n_tokens) break;
            if (sh_base[k] >= 0) {
                uint4 o = w[u];
                if constexpr (Q8) {
                    o.x = q8_value2(__byte_perm(w[u].x, 0, 0x1100), scale[u]);
                    o.y = q8_value2(__byte_perm(w[u].x, 0, 0x3322), scale[u]);
                    o.z = q8_value2(__byte_perm(w[u].z, 0, 0x1100), scale[u]);
                    o.w = q8_value2(__byte_perm(w[u].z, 0, 0x3322), scale[u]);
                }
                const long long to = (t0 + k) * a.out_rs + (r < Hkv ? r : r - Hkv) * D + i0;
                void* out = r < Hkv ? a.k_out : a.v_out;
                if constexpr (F32) {
                    float* dst = static_cast<float*>(out) + to;
                    reinterpret_cast<float4*>(dst)[0] = make_float4(bf16lo(o.x), bf16hi(o.x), bf16lo(o.y), bf16hi(o.y));
                    reinterpret_cast<float4*>(dst)[1] = make_float4(bf16lo(o.z), bf16hi(o.z), bf16lo(o.w), bf16hi(o.w));
                } else {
                    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + to) = o;
                }
            }
            advance(k, r, ROWS, per_token);
        }
    }
}
template <int LPR>
static cudaError_t read_vec_launch(const ReadArgs& a, cudaStream_t st) {
    const int n = tokens_per_block(a.T, a.c.Hkv, LPR);
    if (a.c.scales) return a.f32 ? launch_chained(kv_read_vec_kernel<LPR, true, true>, dim3((a.T + n - 1) / n), dim3(256), 0, st, a, n) : launch_chained(kv_read_vec_kernel<LPR, true, false>, dim3((a.T + n - 1) / n), dim3(256), 0, st, a, n);
    return a.f32 ? launch_chained(kv_read_vec_kernel<LPR, false, true>, dim3((a.T + n - 1) / n), dim3(256), 0, st, a, n) : launch_chained(kv_read_vec_kernel<LPR, false, false>, dim3((a.T + n - 1) / n), dim3(256), 0, st, a, n);
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
    const bool pieces = !((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 15) && kv_row_stride % 8 == 0 && kv_row_stride <= INT32_MAX / (2 * PLACES);
    const int lanes = D <= 64 ? 4 : D <= 128 ? 8 : 16, n = tokens_per_block(T, Hkv, lanes);
    const cudaStream_t st = as_stream(stream);
    const cudaError_t e = !pieces      ? launch_chained(kv_append_q8_kernel, dim3(T), dim3(256), 0, st, a)
                          : lanes == 4 ? append_vec_launch<4>(a, n, st)
                          : lanes == 8 ? append_vec_launch<8>(a, n, st)
                                       : append_vec_launch<16>(a, n, st);
    JSM_CUDA_CHECK(e);
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
