// Quantisation to 8-bit floating point with a scale per block
// (tpk_quant_f8, include/tpmd.h): per block of 1 x 128 or 128 x 128 elements
//   s = max(amax |x| / 448, 2^-126),  q = x / s rounded to e4m3 (nearest even).
// Byte movers: each element is read once into registers, the block's maximum
// formed by shuffles (1 x 128: the lanes that hold the block; 128 x 128: the
// CTA), and written once.
//
// Measured: 16384 x 4096 in 1 x 128 blocks, f16 (203 MB) 39 us, 5.2 TB/s, 0.8
// of the copy rate, f32 (338 MB) 53 us, 6.3 TB/s; 180 x 1024 f32 1.7 us, a
// launch. In 128 x 128 blocks 4096 x 1024 f32 (21 MB) 5.8 us, 3.6 TB/s (256
// CTAs at once: load, maximum and store follow one another), f16 5.5 us;
// 16384 x 4096 f32 82 us, 4.1 TB/s, f16 112 us, 1.8 TB/s (by latency: its warps
// wait for their loads, DRAM 19% busy).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "../../include/tpmd.h"
#include "f8.cuh"
#include "tc_ops.cuh"
#include "tpmd_internal.h"

namespace tpmd {
namespace {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) vec_of {
    T v[VEC];
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// a lane's VEC elements of the block of row `r` that begins at column c0, zero
// from column K on: side by side, or, where rows start off a vector's
// boundary, one in every LANES = 128 / VEC, so that lanes load and store one
// behind the other (3451 x 3663 f16, blocks of 128 x 128: side by side 31 us,
// so 21)
template <typename T, int VEC, bool ALIGNED>
__device__ __forceinline__ vec_of<T, VEC> load_row(const T *r, int64_t c0, int lane, int64_t K) {
    vec_of<T, VEC> x;
    const int64_t c = c0 + lane * (ALIGNED ? VEC : 1);
    constexpr int D = ALIGNED ? 1 : 128 / VEC;
    if (ALIGNED && c + VEC <= K) {
        x = *reinterpret_cast<const vec_of<T, VEC> *>(r + c);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) x.v[e] = c + e * D < K ? r[c + e * D] : T(0.0f);
    }
    return x;
}
// the largest magnitude (NaN does not count)
__device__ __forceinline__ float amax_of(const vec_of<float, 4> &x) {
    return fmaxf(fmaxf(fabsf(x.v[0]), fabsf(x.v[1])), fmaxf(fabsf(x.v[2]), fabsf(x.v[3])));
}
__device__ __forceinline__ __half2 amax2_of(const vec_of<__half, 8> &x) {
    const __half2 *h = reinterpret_cast<const __half2 *>(x.v);
    return __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
}
__device__ __forceinline__ float amax_of(const vec_of<__half, 8> &x) {
    const __half2 a = amax2_of(x);
    return fmaxf(__low2float(a), __high2float(a));
}
// the maxima over the LANES lanes that hold a block, of U blocks
template <int U, int LANES>
__device__ __forceinline__ void amax_lanes(const vec_of<float, 4> (&v)[U], float (&top)[U]) {
#pragma unroll
    for (int u = 0; u < U; u++) {
        top[u] = amax_of(v[u]);
#pragma unroll
        for (int w = LANES / 2; w > 0; w >>= 1) top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], w));
    }
}
// (f16: two blocks' maxima in one register)
template <int U, int LANES>
__device__ __forceinline__ void amax_lanes(const vec_of<__half, 8> (&v)[U], float (&top)[U]) {
#pragma unroll
    for (int u = 0; u < U; u += 2) {
        const __half2 a = amax2_of(v[u]), b = u + 1 < U ? amax2_of(v[u + 1 < U ? u + 1 : u]) : a;
        __half2 t = __hmax2(__lows2half2(a, b), __highs2half2(a, b));
#pragma unroll
        for (int w = LANES / 2; w > 0; w >>= 1) t = __hmax2(t, __shfl_xor_sync(0xffffffffu, t, w));
        top[u] = __low2float(t);
        if (u + 1 < U) top[u + 1] = __high2float(t);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ vec_of<uint8_t, VEC> quant_vec(const vec_of<T, VEC> &x, f8_scale s) {
    vec_of<uint8_t, VEC> t;
#pragma unroll
    for (int e = 0; e < VEC; e += 4)
        *reinterpret_cast<uint32_t *>(t.v + e) = f8_quant4(to_f(x.v[e]), to_f(x.v[e + 1]), to_f(x.v[e + 2]), to_f(x.v[e + 3]), s);
    return t;
}
template <typename T, int VEC, bool ALIGNED>
__device__ __forceinline__ void store_row(uint8_t *r, int64_t c0, int lane, int64_t K, f8_scale s,
                                          const vec_of<T, VEC> &x) {
    const vec_of<uint8_t, VEC> t = quant_vec(x, s);
    const int64_t c = c0 + lane * (ALIGNED ? VEC : 1);
    constexpr int D = ALIGNED ? 1 : 128 / VEC;
    if (ALIGNED && c + VEC <= K) {
        *reinterpret_cast<vec_of<uint8_t, VEC> *>(r + c) = t;
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e++)
            if (c + e * D < K) r[c + e * D] = t.v[e];
    }
}

// rows = 1: 128 / VEC lanes hold a block, VEC elements (16 bytes) each; a warp
// takes GROUP blocks of a row at a time, all their loads in flight together
template <typename T, int VEC, bool ALIGNED, int U>
__global__ void __launch_bounds__(256) quant_rows_kernel(const T *x, int64_t ldx, int64_t M, int64_t K,
                                                         int kb, uint8_t *__restrict__ q, int64_t ldq,
                                                         float *__restrict__ s, int64_t lds) {
    pdl_wait();
    pdl_trigger();
    constexpr int LANES = 128 / VEC, GROUP = U * 32 / LANES;
    const int per_row = (kb + GROUP - 1) / GROUP, lane = threadIdx.x % LANES, sub = threadIdx.x % 32 / LANES;
    const int64_t warps = (int64_t) gridDim.x * 8, w0 = (int64_t) blockIdx.x * 8 + threadIdx.x / 32;
    // (row, group of blocks), advanced without a division
    int64_t m = w0 / per_row;
    int g = (int) (w0 % per_row);
    const int64_t dm = warps / per_row;
    const int dg = (int) (warps % per_row);
    for (; m < M; m += dm, g += dg) {
        if (g >= per_row) {
            g -= per_row;
            if (++m >= M) break;
        }
        vec_of<T, VEC> v[U];
        float top[U];
        constexpr int STEP = 32 / LANES * 128;  // columns a load of a warp
        const int64_t c0 = ((int64_t) g * GROUP + sub) * 128, c = c0 + lane * VEC;
        if (ALIGNED && (int64_t) (g + 1) * GROUP * 128 <= K) {  // whole blocks: no column to look at
            const T *xp = x + m * ldx + c;
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = *reinterpret_cast<const vec_of<T, VEC> *>(xp + u * STEP);
            amax_lanes<U, LANES>(v, top);
            uint8_t *qp = q + m * ldq + c;
            float *sp = s + m * lds + g * GROUP + sub;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const f8_scale sc = f8_scale_of(top[u]);
                *reinterpret_cast<vec_of<uint8_t, VEC> *>(qp + u * STEP) = quant_vec(v[u], sc);
                if (lane == 0) sp[u * (STEP / 128)] = sc.s;
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = load_row<T, VEC, ALIGNED>(x + m * ldx, c0 + u * STEP, lane, K);
            amax_lanes<U, LANES>(v, top);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int b = g * GROUP + u * (32 / LANES) + sub;
                const f8_scale sc = f8_scale_of(top[u]);
                if (b < kb) {
                    store_row<T, VEC, ALIGNED>(q + m * ldq, c0 + u * STEP, lane, K, sc, v[u]);
                    if (lane == 0) s[m * lds + b] = sc.s;
                }
            }
        }
    }
}

// rows = 128: a CTA holds the 128 x 128 block, 64 elements a thread
template <typename T, int VEC, bool ALIGNED>
__global__ void __launch_bounds__(256) quant_blocks_kernel(const T *x, int64_t ldx, int64_t M, int64_t K,
                                                           int64_t kb, uint8_t *__restrict__ q, int64_t ldq,
                                                           float *__restrict__ s, int64_t lds) {
    pdl_wait();
    pdl_trigger();
    constexpr int LANES = 128 / VEC, ROWS = 256 / LANES, N = 128 / ROWS;
    __shared__ float red[8];
    const int64_t mb = blockIdx.x / kb, b = blockIdx.x % kb;
    const int64_t c0 = b * 128, r0 = mb * 128 + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    vec_of<T, VEC> v[N];
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int64_t m = r0 + i * ROWS;
        // rows behind the last one load as zeros (no column below 0)
        v[i] = load_row<T, VEC, ALIGNED>(x + (m < M ? m : 0) * ldx, c0, lane, m < M ? K : 0);
        a = fmaxf(a, amax_of(v[i]));
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
        if (r0 + i * ROWS < M) store_row<T, VEC, ALIGNED>(q + (r0 + i * ROWS) * ldq, c0, lane, K, sc, v[i]);
    if (threadIdx.x == 0) s[mb * lds + b] = sc.s;
}

template <typename T, int VEC, bool ALIGNED>
cudaError_t run_quant(const void *x, int64_t ldx, int64_t M, int64_t K, int rows, void *q, int64_t ldq, float *s,
                      int64_t lds, cudaStream_t st) {
    const int64_t kb = (K + 127) / 128;
    if (rows == 1) {
        // loads in flight a lane: four where the blocks fill the SMs' warps all
        // the same, else one (180 x 1024 f32: 2.0 us, with four 3.1)
        auto go = [&](auto kernel, int group) {
            const int64_t ctas = (M * ((kb + group - 1) / group) + 7) / 8;
            const dim3 grid((unsigned) std::min<int64_t>(ctas, sm_count() * 8));
            return launch_pdl(kernel, grid, dim3(256), 0, st, (const T *) x, ldx, M, K, (int) kb, (uint8_t *) q, ldq, s,
                              lds);
        };
        constexpr int PER = VEC / 4;  // blocks a load of a warp
        if (M * ((kb + 4 * PER - 1) / (4 * PER)) >= sm_count() * 64) return go(quant_rows_kernel<T, VEC, ALIGNED, 4>, 4 * PER);
        return go(quant_rows_kernel<T, VEC, ALIGNED, 1>, PER);
    }
    const int64_t ctas = (M + 127) / 128 * kb;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    return launch_pdl(quant_blocks_kernel<T, VEC, ALIGNED>, dim3((unsigned) ctas), dim3(256), 0, st, (const T *) x, ldx, M,
                      K, kb, (uint8_t *) q, ldq, s, lds);
}

}  // namespace

cudaError_t quant_f8(const void *x, bool f16, int64_t ldx, int64_t M, int64_t K, int rows, void *q, int64_t ldq, float *s,
                     int64_t lds, cudaStream_t st) {
    const int es = f16 ? 2 : 4, vec = 16 / es;
    // whole 16-byte loads and 4- or 8-byte stores where every row starts aligned for them
    const bool al = !((uintptr_t) x & 15) && !((uintptr_t) q & (vec - 1)) &&
                    (M == 1 || (ldx * es % 16 == 0 && ldq % vec == 0));
    if (f16)
        return al ? run_quant<__half, 8, true>(x, ldx, M, K, rows, q, ldq, s, lds, st)
                  : run_quant<__half, 8, false>(x, ldx, M, K, rows, q, ldq, s, lds, st);
    return al ? run_quant<float, 4, true>(x, ldx, M, K, rows, q, ldq, s, lds, st)
              : run_quant<float, 4, false>(x, ldx, M, K, rows, q, ldq, s, lds, st);
}

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
    const cudaError_t e = quant_f8(x, dtype == TPMD_DTYPE_F16, ldx, M, K, rows, q, ldq, s, lds, (cudaStream_t) stream);
    if (e == cudaErrorInvalidValue) return fail("too many blocks");
    if (e != cudaSuccess) return fail(cudaGetErrorString(e));
    return 0;
}

extern "C" int tpk_quant_f8_packed(const int64_t args[11]) {
    tpmd::packed_args p{args};
    const void *x = p.ptr();
    const int dtype = p.i32();
    const int64_t ldx = p.i64(), M = p.i64(), K = p.i64();
    const int rows = p.i32();
    void *q = p.ptr();
    const int64_t ldq = p.i64();
    float *s = (float *) p.ptr();
    const int64_t lds = p.i64();
    void *stream = p.ptr();
    if (!p.fits) return tpmd::tpk_fail("tpk_quant_f8: an argument is out of its range");
    return tpk_quant_f8(x, dtype, ldx, M, K, rows, q, ldq, s, lds, stream);
}
