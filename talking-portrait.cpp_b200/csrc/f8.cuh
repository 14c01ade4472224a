// Quantisation to e4m3 with a scale per block, shared by tpk_quant_f8 and
// the 8-bit output of tpk_gemm_f8:
//   s = max(amax / 448, 2^-126),  q = x / s rounded to e4m3 (nearest even)
// in IEEE float32.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace tpmd {
namespace {

struct f8_scale {
    float s;
    float r;  // 1 / s, or 0 where the quotient takes the IEEE division
};
__device__ __forceinline__ f8_scale f8_scale_of(float amax) {
    f8_scale k;
    k.s = fmaxf(__fdiv_rn(amax, 448.0f), 1.17549435e-38f);
    // 2^-90 .. 2^120: the reciprocal and the remainders that matter are normal numbers
    k.r = k.s >= 8.07793567e-28f && k.s <= 1.32922800e+36f ? __frcp_rn(k.s) : 0.0f;
    return k;
}
// x / s: a product with the reciprocal and one correction by the exact
// remainder (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990): within 2^-46 of the quotient before its last
// rounding, so the same float32 as the division's; four instructions
// where that takes a dozen and a branch
__device__ __forceinline__ float f8_quotient(float x, f8_scale k) {
    const float q = x * k.r;
    return copysignf(fmaf(fmaf(-q, k.s, x), k.r, q), x);  // (a zero keeps its sign)
}
// four elements as bytes, the first lowest
__device__ __forceinline__ uint32_t f8_quant4(float a, float b, float c, float d, f8_scale k) {
    if (k.r != 0.0f) {
        a = f8_quotient(a, k);
        b = f8_quotient(b, k);
        c = f8_quotient(c, k);
        d = f8_quotient(d, k);
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
