// Rotary positions on the query and key heads of token rows of any pitch: adjacent pairs or halves, on the first rot_dim components of a head, from
// the (cos, sin) tables of jsm_rope_half_table / jsm_rope_scaled_table; transposed, it is the gradient of the rotation.
//   pair (x1, x2) -> (x1 c - x2 s, x2 c + x1 s),  transposed: s -> -s
// Bound by memory: every row is read and written once.  The table (8 bytes per pair, twice the bytes of a bf16 pair) would cost more than one head, so a thread keeps
// the entries of its eight (fp32: four) pairs and walks the heads with them.
#include "cache_view.cuh"

namespace jsm {

int* tc_error_word();

struct RotateArgs {
    const void *q, *k;
    void *q_out, *k_out;
    long long q_rs, k_rs, qo_rs, ko_rs;  // row pitches, elements
    int Hq, Hk, D, rot, adjacent;
    float sign;                          // -1: transposed
    const float2* table;
    int table_len;
    const int32_t* positions;
    int T;
    int* err;
};

template <typename T>
__device__ __forceinline__ float rot_load(const T* p);
template <>
__device__ __forceinline__ float rot_load<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float rot_load<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void rot_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void rot_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// any sizes, pitches and alignments: a thread has a pair or an unrotated component, and walks the heads with its table entry
template <typename T>
__global__ void __launch_bounds__(256) rope_rotate_scalar_kernel(RotateArgs a) {
    chain_trigger();
    chain_wait();
    const int half = a.rot / 2, units = a.D - half, heads = a.Hq + a.Hk, head_lanes = max(1, 256 / units);
    const int u0 = units < 256 ? threadIdx.x % units : threadIdx.x, hl = units < 256 ? threadIdx.x / units : 0;
    if (hl >= head_lanes) return;
    const int t = blockIdx.x, pos = a.positions ? a.positions[t] : t;
    if (pos < 0 || pos >= a.table_len) {
        if (threadIdx.x == 0) cache_error(a.err, CACHE_BAD_POSITION);
        return;
    }
    for (int u = u0; u < units; u += 256) {
        const float2 e = u < half ? a.table[(long long)pos * half + u] : make_float2(0.0f, 0.0f);
        const int i1 = u < half ? (a.adjacent ? 2 * u : u) : u + half, i2 = a.adjacent ? 2 * u + 1 : u + half;
        for (int h = hl; h < heads; h += head_lanes) {
            const bool is_q = h < a.Hq;
            const T* src = is_q ? static_cast<const T*>(a.q) + t * a.q_rs + (long long)h * a.D : static_cast<const T*>(a.k) + t * a.k_rs + (long long)(h - a.Hq) * a.D;
            T* dst = is_q ? static_cast<T*>(a.q_out) + t * a.qo_rs + (long long)h * a.D : static_cast<T*>(a.k_out) + t * a.ko_rs + (long long)(h - a.Hq) * a.D;
            if (u < half) {
                float y1, y2;
                rotate_pair(rot_load(src + i1), rot_load(src + i2), e.x, a.sign * e.y, y1, y2);
                rot_store(dst + i1, y1);
                rot_store(dst + i2, y2);
            } else {
                dst[i1] = src[i1];
            }
        }
    }
}

// Whole 16-byte pieces: a thread has one unit of a head - a piece of each half, a piece of adjacent pairs, or a piece that is not rotated - with its table entries in
// registers, and takes that unit of every HL-th head, four heads' loads in flight.  8192 rows of 32 + 8 heads of 128 with 64 rotated (bf16, 170 MB): 32.3 us, 5.3 TB/s of the
// measured 6.5, with seven blocks per multiprocessor (six 33.5, ten spill: 46); without streaming loads and stores 36.1, with position and table ahead of the rows 40.7.
template <typename T>
struct RotPiece {
    static constexpr int V = 16 / sizeof(T);
    float x[V];
    __device__ __forceinline__ void unpack(const uint4& w) {
        const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) {
                x[2 * i] = bf16lo(in[i]);
                x[2 * i + 1] = bf16hi(in[i]);
            } else {
                x[i] = __uint_as_float(in[i]);
            }
        }
    }
    __device__ __forceinline__ uint4 pack() const {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) o[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
            else o[i] = __float_as_uint(x[i]);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};

constexpr int RV_THREADS = 128;
template <typename T, bool ADJACENT>
__global__ void __launch_bounds__(RV_THREADS, 7) rope_rotate_vec_kernel(RotateArgs a, int units, int head_lanes) {
    constexpr int V = RotPiece<T>::V, PAIRS = ADJACENT ? V / 2 : V, U = 4;
    chain_trigger();
    chain_wait();
    const int u = threadIdx.x % units, hl = threadIdx.x / units, heads = a.Hq + a.Hk;
    if (hl >= head_lanes) return;
    const int rotated = (ADJACENT ? a.rot : a.rot / 2) / V;      // units that are
    const int first = (ADJACENT || u < rotated ? u : u + rotated) * V;  // component of the unit's (first) piece
    const int t = blockIdx.x, half = a.rot / 2;
    const T *q = static_cast<const T*>(a.q) + t * a.q_rs + first, *k = static_cast<const T*>(a.k) + t * a.k_rs + first;
    T *qo = static_cast<T*>(a.q_out) + t * a.qo_rs + first, *ko = static_cast<T*>(a.k_out) + t * a.ko_rs + first;
    uint4 w[U], w2[U];
    auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int h = h0 + i * head_lanes;
            if (h >= heads) break;
            const T* src = h < a.Hq ? q + (long long)h * a.D : k + (long long)(h - a.Hq) * a.D;
            w[i] = __ldcs(reinterpret_cast<const uint4*>(src));
            if (!ADJACENT && u < rotated) w2[i] = __ldcs(reinterpret_cast<const uint4*>(src + half));
        }
    };
    load(hl);  // (before position and table: one latency of three in a row)
    const int pos = a.positions ? a.positions[t] : t;
    if (pos < 0 || pos >= a.table_len) {
        if (threadIdx.x == 0) cache_error(a.err, CACHE_BAD_POSITION);
        return;
    }
    float c[PAIRS], s[PAIRS];
    if (u < rotated) {
        const float4* e = reinterpret_cast<const float4*>(a.table + (long long)pos * half + u * PAIRS);
#pragma unroll
        for (int i = 0; i < PAIRS / 2; ++i) {
            const float4 v = e[i];
            c[2 * i] = v.x; s[2 * i] = a.sign * v.y; c[2 * i + 1] = v.z; s[2 * i + 1] = a.sign * v.w;
        }
    }
    for (int h0 = hl; h0 < heads; h0 += U * head_lanes) {
        if (h0 != hl) load(h0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int h = h0 + i * head_lanes;
            if (h >= heads) break;
            T* dst = h < a.Hq ? qo + (long long)h * a.D : ko + (long long)(h - a.Hq) * a.D;
            if (u < rotated) {
                RotPiece<T> x, y;
                x.unpack(w[i]);
                if constexpr (ADJACENT) {
#pragma unroll
                    for (int n = 0; n < PAIRS; ++n) rotate_pair(x.x[2 * n], x.x[2 * n + 1], c[n], s[n], x.x[2 * n], x.x[2 * n + 1]);
                } else {
                    y.unpack(w2[i]);
#pragma unroll
                    for (int n = 0; n < PAIRS; ++n) rotate_pair(x.x[n], y.x[n], c[n], s[n], x.x[n], y.x[n]);
                    __stcs(reinterpret_cast<uint4*>(dst + half), y.pack());
                }
                w[i] = x.pack();
            }
            __stcs(reinterpret_cast<uint4*>(dst), w[i]);
        }
    }
}

template <typename T>
static jsm_status rotate_vec_launch(const RotateArgs& a, cudaStream_t st) {
    constexpr int V = RotPiece<T>::V;
    const int units = a.adjacent ? a.D / V : a.D / V - a.rot / 2 / V, heads = a.Hq + a.Hk;
    const int head_lanes = RV_THREADS / units < heads ? RV_THREADS / units : heads;
    JSM_CUDA_CHECK(a.adjacent ? launch_chained(rope_rotate_vec_kernel<T, true>, dim3(a.T), dim3(units * head_lanes), 0, st, a, units, head_lanes)
                              : launch_chained(rope_rotate_vec_kernel<T, false>, dim3(a.T), dim3(units * head_lanes), 0, st, a, units, head_lanes));
    JSM_LAUNCH_CHECK();
    return JSM_OK;
}

}  // namespace jsm

using namespace jsm;

extern "C" jsm_status jsm_rope_rotate(const void* d_q, int64_t q_row_stride, void* d_q_out, int64_t q_out_row_stride, int Hq, const void* d_k, int64_t k_row_stride,
                                      void* d_k_out, int64_t k_out_row_stride, int Hkv, jsm_dtype dtype, int D, const float* d_table, int table_len, int rot_dim,
                                      int layout, int transposed, const int32_t* d_positions, int T, void* stream) {
    if (T < 0 || Hq < 0 || Hkv < 0 || Hq + (int64_t)Hkv > INT32_MAX / 4) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: T %d, heads %d and %d", T, Hq, Hkv);
    if (D <= 0 || D > 4096 || rot_dim <= 0 || rot_dim % 2 || rot_dim > D) JSM_FAIL(JSM_SHAPE, "jsm_rope_rotate: rotation of %d components of a head of %d", rot_dim, D);
    if ((Hq + (int64_t)Hkv) * D > INT32_MAX) JSM_FAIL(JSM_SHAPE, "jsm_rope_rotate: heads %d and %d of %d", Hq, Hkv, D);
    if (layout != JSM_ROPE_ADJACENT && layout != JSM_ROPE_HALF) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: layout %d", layout);
    if (dtype != JSM_F32 && dtype != JSM_BF16) JSM_FAIL(JSM_UNSUPPORTED, "jsm_rope_rotate: dtype %d", (int)dtype);
    if (table_len <= 0) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: a table of %d positions", table_len);
    if (T == 0 || Hq + Hkv == 0) return JSM_OK;
    if (!d_table || (Hq > 0 && (!d_q || !d_q_out)) || (Hkv > 0 && (!d_k || !d_k_out))) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: null pointer");
    if (Hq > 0 && (q_row_stride < (int64_t)Hq * D || q_out_row_stride < (int64_t)Hq * D)) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: query rows overlap");
    if (Hkv > 0 && (k_row_stride < (int64_t)Hkv * D || k_out_row_stride < (int64_t)Hkv * D)) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: key rows overlap");
    if (reinterpret_cast<uintptr_t>(d_table) & 7) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: the table is not 8-byte aligned");
    const uintptr_t odd = reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_q_out) | reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_k_out);
    if (odd & (dtype == JSM_F32 ? 3 : 1)) JSM_FAIL(JSM_INVALID_ARG, "jsm_rope_rotate: rows that are not aligned to their elements");
    RotateArgs a{d_q, d_k, d_q_out, d_k_out, q_row_stride, k_row_stride, q_out_row_stride, k_out_row_stride, Hq, Hkv, D, rot_dim, layout == JSM_ROPE_ADJACENT ? 1 : 0,
                 transposed ? -1.0f : 1.0f, reinterpret_cast<const float2*>(d_table), table_len, d_positions, T, tc_error_word()};
    const int V = dtype == JSM_F32 ? 4 : 8;
    const int64_t pitches = (Hq ? q_row_stride | q_out_row_stride : 0) | (Hkv ? k_row_stride | k_out_row_stride : 0);
    if (!((odd | reinterpret_cast<uintptr_t>(d_table)) & 15) && pitches % V == 0 && D % V == 0 && (layout == JSM_ROPE_ADJACENT ? rot_dim : rot_dim / 2) % V == 0 && D / V <= RV_THREADS)
        return dtype == JSM_F32 ? rotate_vec_launch<float>(a, as_stream(stream)) : rotate_vec_launch<__nv_bfloat16>(a, as_stream(stream));
    const dim3 grid(T);
    if (dtype == JSM_F32) JSM_CUDA_CHECK(launch_chained(rope_rotate_scalar_kernel<float>, grid, dim3(256), 0, as_stream(stream), a));
    else JSM_CUDA_CHECK(launch_chained(rope_rotate_scalar_kernel<__nv_bfloat16>, grid, dim3(256), 0, as_stream(stream), a));
    JSM_LAUNCH_CHECK();
    return JSM_OK;
}
