// Quantisation to 8-bit floating point with a scale per block
// (tpk_quant_f8, include/tpmd.h): per block of 1 x 128 or 128 x 128 elements
//   s = max(amax |x| / 448, 2^-126),  q = x / s rounded to e4m3 (nearest even).
// Byte movers: each element is read once into registers, the block's maximum
// formed by shuffles (1 x 128: the lanes that hold the block; 128 x 128: the
// CTA), and written once.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "../../include/tpmd.h"
#include "f8.cuh"
#include "tpmd_internal.h"

namespace tpmd {
namespace {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) vec_of {
    T v[VEC];
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// VEC elements of row `r` from column c, zero from column K on
template <typename T, int VEC, bool ALIGNED>
__device__ __forceinline__ void load_row(const T *r, int64_t c, int64_t K, float (&x)[VEC]) {
    if (ALIGNED && c + VEC <= K) {
        const vec_of<T, VEC> t = *reinterpret_cast<const vec_of<T, VEC> *>(r + c);
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = to_f(t.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = c + e < K ? to_f(r[c + e]) : 0.0f;
    }
}
template <int VEC, bool ALIGNED>
__device__ __forceinline__ void store_row(uint8_t *r, int64_t c, int64_t K, f8_scale s, const float (&x)[VEC]) {
    vec_of<uint8_t, VEC> t;
#pragma unroll
    for (int e = 0; e < VEC; e += 4)
        *reinterpret_cast<uint32_t *>(t.v + e) = f8_quant4(x[e], x[e + 1], x[e + 2], x[e + 3], s);
    if (ALIGNED && c + VEC <= K) {
        *reinterpret_cast<vec_of<uint8_t, VEC> *>(r + c) = t;
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e++)
            if (c + e < K) r[c + e] = t.v[e];
    }
}

// rows = 1: 128 / VEC lanes hold a block, VEC elements (16 bytes) each
template <typename T, int VEC, bool ALIGNED>
__global__ void __launch_bounds__(256) quant_rows_kernel(const T *__restrict__ x, int64_t ldx, int64_t M, int64_t K,
                                                         int64_t kb, uint8_t *__restrict__ q, int64_t ldq,
                                                         float *__restrict__ s, int64_t lds) {
    constexpr int LANES = 128 / VEC;
    const int64_t nblk = M * kb, per = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    for (int64_t blk = (int64_t) blockIdx.x * per + threadIdx.x / LANES; blk < nblk; blk += (int64_t) gridDim.x * per) {
        const int64_t m = blk / kb, b = blk % kb, c = b * 128 + lane * VEC;
        float v[VEC], a = 0.0f;
        load_row<T, VEC, ALIGNED>(x + m * ldx, c, K, v);
#pragma unroll
        for (int e = 0; e < VEC; e++) a = fmaxf(a, fabsf(v[e]));
        const unsigned mask = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
#pragma unroll
        for (int w = LANES / 2; w > 0; w >>= 1) a = fmaxf(a, __shfl_xor_sync(mask, a, w));
        const f8_scale sc = f8_scale_of(a);
        store_row<VEC, ALIGNED>(q + m * ldq, c, K, sc, v);
        if (lane == 0) s[m * lds + b] = sc.s;
    }
}

// rows = 128: a CTA holds the 128 x 128 block, 64 elements a thread
template <typename T, int VEC, bool ALIGNED>
__global__ void __launch_bounds__(256) quant_blocks_kernel(const T *__restrict__ x, int64_t ldx, int64_t M, int64_t K,
                                                           int64_t kb, uint8_t *__restrict__ q, int64_t ldq,
                                                           float *__restrict__ s, int64_t lds) {
    constexpr int LANES = 128 / VEC, ROWS = 256 / LANES, N = 128 / ROWS;
    __shared__ float red[8];
    const int64_t mb = blockIdx.x / kb, b = blockIdx.x % kb;
    const int64_t c = b * 128 + threadIdx.x % LANES * VEC, r0 = mb * 128 + threadIdx.x / LANES;
    float v[N][VEC], a = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int64_t m = r0 + i * ROWS;
        // rows behind the last one load as zeros (no column below 0)
        load_row<T, VEC, ALIGNED>(x + (m < M ? m : 0) * ldx, c, m < M ? K : 0, v[i]);
#pragma unroll
        for (int e = 0; e < VEC; e++) a = fmaxf(a, fabsf(v[i][e]));
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, w));
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) a = fmaxf(a, red[w]);
    const f8_scale sc = f8_scale_of(a);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (r0 + i * ROWS < M) store_row<VEC, ALIGNED>(q + (r0 + i * ROWS) * ldq, c, K, sc, v[i]);
    if (threadIdx.x == 0) s[mb * lds + b] = sc.s;
}

template <typename T, int VEC, bool ALIGNED>
cudaError_t run_quant(const void *x, int64_t ldx, int64_t M, int64_t K, int rows, void *q, int64_t ldq, float *s,
                      int64_t lds, cudaStream_t st) {
    const int64_t kb = (K + 127) / 128;
    if (rows == 1) {
        const int64_t ctas = (M * kb + 2 * VEC - 1) / (2 * VEC);
        quant_rows_kernel<T, VEC, ALIGNED><<<(unsigned) std::min<int64_t>(ctas, 148 * 64), 256, 0, st>>>(
            (const T *) x, ldx, M, K, kb, (uint8_t *) q, ldq, s, lds);
    } else {
        const int64_t ctas = (M + 127) / 128 * kb;
        if (ctas > INT32_MAX) return cudaErrorInvalidValue;
        quant_blocks_kernel<T, VEC, ALIGNED><<<(unsigned) ctas, 256, 0, st>>>(
            (const T *) x, ldx, M, K, kb, (uint8_t *) q, ldq, s, lds);
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace tpmd

extern "C" int tpk_quant_f8(const void *x, int dtype, int64_t ldx, int64_t M, int64_t K, int rows, void *q,
                            int64_t ldq, float *s, int64_t lds, void *stream) {
    using namespace tpmd;
    auto fail = [](const char *m) { return tpk_fail(std::string("tpk_quant_f8: ") + m); };
    if (dtype != TPMD_DTYPE_F32 && dtype != TPMD_DTYPE_F16) return fail("dtype");
    if (rows != 1 && rows != 128) return fail("rows must be 1 or 128");
    if (M < 0 || K < 0 || M >= 1ll << 40 || K >= 1ll << 31) return fail("bad shape");
    if (M == 0 || K == 0) return 0;
    if (!x || !q || !s) return fail("null pointer");
    if ((M > 1 && (ldx < 0 || ldq < K)) || (M > rows && lds < (K + 127) / 128)) return fail("bad row stride");
    if ((uintptr_t) x & (dtype == TPMD_DTYPE_F16 ? 1 : 3) || (uintptr_t) s & 3)
        return fail("a pointer is not aligned to its element type");
    const void *ptrs[] = {x, q, s};
    tpk_device_scope dev(ptrs, 3);
    if (!dev.ok()) return fail(dev.why);
    const bool f16 = dtype == TPMD_DTYPE_F16;
    const int es = f16 ? 2 : 4, vec = 16 / es;
    // whole 16-byte loads and 4- or 8-byte stores where every row starts aligned for them
    const bool al = !((uintptr_t) x & 15) && !((uintptr_t) q & (vec - 1)) &&
                    (M == 1 || (ldx * es % 16 == 0 && ldq % vec == 0));
    cudaStream_t st = (cudaStream_t) stream;
    cudaError_t e;
    if (f16)
        e = al ? run_quant<__half, 8, true>(x, ldx, M, K, rows, q, ldq, s, lds, st)
               : run_quant<__half, 8, false>(x, ldx, M, K, rows, q, ldq, s, lds, st);
    else
        e = al ? run_quant<float, 4, true>(x, ldx, M, K, rows, q, ldq, s, lds, st)
               : run_quant<float, 4, false>(x, ldx, M, K, rows, q, ldq, s, lds, st);
    if (e == cudaErrorInvalidValue) return fail("too many blocks");
    if (e != cudaSuccess) return fail(cudaGetErrorString(e));
    return 0;
}
