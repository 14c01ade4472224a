// Quantisation to e4m3 with a scale per block, shared by tpk_quant_f8 and
// the 8-bit output of tpk_gemm_f8:
//   s = max(amax / 448, 2^-126),  q = x / s rounded to e4m3 (nearest even)
// in float32.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace tpmd {
namespace {

// A quotient takes a product with the reciprocal and one correction by the
// exact remainder (Markstein, "Computation of elementary functions on the IBM
// RISC System/6000 processor", 1990): within 2^-44 of the quotient before
// its last rounding, so the same float32 as the division's unless that lies
// as near to a rounding border; 1.5 packed instructions an element where the
// division takes a dozen and a branch. (Of a zero's sign nothing is kept.)
struct f8_scale {
    float s;
    float r;  // 1 / s within an ulp, or 0 where the quotient takes the IEEE division
};
__device__ __forceinline__ f8_scale f8_scale_of(float amax) {
    amax = fmaxf(amax, 0.0f);  // (of a block of nothing but NaN: none of them counts)
    // amax / 448 the same way; an infinite maximum stays
    constexpr float R448 = 1.0f / 448.0f;
    const float q = amax * R448;
    f8_scale k;
    k.s = amax <= 3.4028235e38f ? fmaxf(fmaf(fmaf(-q, 448.0f, amax), R448, q), 1.17549435e-38f) : amax;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(k.s));
    // 2^-90 .. 2^120: the reciprocal and the remainders that matter are normal numbers
    // (zeros are zeros, and NaN NaN, times any number; padding is made of them)
    k.r = amax == 0.0f ? 1.0f : k.s >= 8.07793567e-28f && k.s <= 1.32922800e+36f ? r : 0.0f;
    return k;
}
// two elements' quotients
__device__ __forceinline__ void f8_quotients(float &a, float &b, f8_scale k) {
    asm("{\n\t.reg .b64 x, r, s, q, e;\n\t"
        "mov.b64 x, {%0, %1};\n\t"
        "mov.b64 r, {%2, %2};\n\t"
        "mov.b64 s, {%3, %3};\n\t"
        "mul.rn.f32x2 q, x, r;\n\t"
        "fma.rn.f32x2 e, q, s, x;\n\t"
        "fma.rn.f32x2 q, e, r, q;\n\t"
        "mov.b64 {%0, %1}, q;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(k.r), "f"(-k.s));
}
// four elements as bytes, the first lowest
__device__ __forceinline__ uint32_t f8_quant4(float a, float b, float c, float d, f8_scale k) {
    if (k.r != 0.0f) {
        f8_quotients(a, b, k);
        f8_quotients(c, d, k);
    } else {
        a = __fdiv_rn(a, k.s);
        b = __fdiv_rn(b, k.s);
        c = __fdiv_rn(c, k.s);
        d = __fdiv_rn(d, k.s);
    }
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return lo | (uint32_t) hi << 16;
}

}  // namespace
}  // namespace tpmd
