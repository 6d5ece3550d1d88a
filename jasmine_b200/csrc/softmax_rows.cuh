// Arithmetic of softmax rows held in registers: base-2 exponentials on both pipes, packed fp32 pairs.
#pragma once
#include "common.cuh"

namespace jsm {

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Blackwell's packed fp32 pairs and three-input maximum: half the FMA / ADD / MAX instructions of the softmax rows
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^x for a pair of scores without the special-function unit: x = n + f with n = round(x) taken from the mantissa of
// x + 1.5 * 2^23, 2^f on [-0.5, 0.5] by a cubic (relative error 7.5e-5, far below the bf16 rounding of P), n added to
// the exponent field.  The MUFU pipe (16 results per clock and SM) is what the softmax of a tile waits for once the
// tensor pipe runs tcgen05 rates, so a share of the exponentials goes to the FMA pipe instead.
__device__ __forceinline__ void ex2_poly2(uint64_t x2, float& p0, float& p1) {
    float x0, x1;
    unpack2(x2, x0, x1);
    x2 = pack2(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
    const uint64_t magic2 = pack2(12582912.0f, 12582912.0f), neg_magic2 = pack2(-12582912.0f, -12582912.0f);
    const uint64_t r2 = fadd2(x2, magic2);
    const uint64_t n2 = fadd2(r2, neg_magic2);
    const uint64_t f2 = ffma2(n2, pack2(-1.0f, -1.0f), x2);
    uint64_t q2 = ffma2(pack2(0.0551716685f, 0.0551716685f), f2, pack2(0.2426111251f, 0.2426111251f));
    q2 = ffma2(q2, f2, pack2(0.6932609677f, 0.6932609677f));
    q2 = ffma2(q2, f2, pack2(0.9999280572f, 0.9999280572f));
    float q0, q1, r0, r1;
    unpack2(q2, q0, q1);
    unpack2(r2, r0, r1);
    p0 = __int_as_float(__float_as_int(q0) + (__float_as_int(r0) << 23));
    p1 = __int_as_float(__float_as_int(q1) + (__float_as_int(r1) << 23));
}

}  // namespace jsm
