// The product of two block-quantised 8-bit matrices on the tcgen05 tensor
// cores (tpk_gemm_f8, include/tpmd.h):
//
//   Y[m][n] = act( sum_b sx[m][b] sw[n/128][b] P_b[m][n] + bias[n] ),
//   P_b[m][n] = sum_{k in block b} X[m][k] W[n][k],  blocks of 128 along k
//
// A CTA owns a 128 x 128 output tile: 128 rows of X are the MMA's M side
// (TMEM lanes), one block of 128 rows of W its N side, so all of a tile's
// W scales of one k block are one number and a lane's factor sx sw is one
// number for all its columns. Each k block of 128 is one pipeline stage (one
// 128-byte swizzled row a matrix row) and one MMA group into an accumulator
// of its own out of a ring in TMEM; eight warps read it (each a lane
// quarter and half of the columns), scale it and add it to f32 registers
// while the next blocks multiply. The products of e4m3 values are exact in
// f32; sums are f32 throughout.
//
// Every pipeline wait is bounded; an expired wait sets *err and the CTA
// skips the rest of its work.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tc_ptx.cuh"
#include "tpmd_internal.h"
#include "../../include/tpmd.h"

#include <algorithm>
#include <cstring>
#include <mutex>
#include <string>

namespace tpmd {
namespace {

constexpr float F8_MAX = 448.0f;
constexpr float S_MIN = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    const uint32_t mask = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(mask));
}

__device__ __forceinline__ float act_fn(float v, int act) {
    if (act == 1) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    if (act == 2) return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
    if (act == 3) return fmaxf(v, 0.2f * v);
    return v;
}

struct f8_cfg {
    static constexpr int BM = 128, BN = 128, KB = 128;
    static constexpr int A_BYTES = BM * KB, B_BYTES = BN * KB, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = 6, NACC = 4;
    static constexpr uint32_t TMEM_COLS = NACC * BN;
    // D f32 (bit 4); A and B e4m3 (0 at bits 7 and 10); K-major both; N >> 3 at bit 17; M >> 4 at bit 24
    static constexpr uint32_t IDESC = (1u << 4) | ((uint32_t) (BN >> 3) << 17) | ((uint32_t) (BM >> 4) << 24);
    static constexpr int NEPI = 8, THREADS = 64 + 32 * NEPI;
    static constexpr int NBARS = 2 * STAGES + 2 * NACC;
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + NBARS * 8 + 16;
    static_assert(SMEM <= 232448, "shared memory");
};

struct f8_params {
    int M, N, K, kblocks, tiles_n;
    const float *sx, *sw, *bias;
    int64_t ldsx, ldsw;
    void *Y;
    int64_t ldy;
    float *sy;
    int64_t ldsy;
    int act;
    bool y_vec;  // Y takes 16-byte stores
    int *err;
};

// N values of one row to Y columns [n, n + CNT)
template <typename TY, int CNT>
__device__ __forceinline__ void store_cols(TY *y, const TY (&v)[CNT], int n, int N, bool vec) {
    constexpr int PER = 16 / sizeof(TY);
#pragma unroll
    for (int c = 0; c < CNT; c += PER) {
        if (vec && n + c + PER <= N) {
            *reinterpret_cast<uint4 *>(y + n + c) = *reinterpret_cast<const uint4 *>(v + c);
        } else {
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (n + c + e < N) y[n + c + e] = v[c + e];
        }
    }
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// AND of v over the epilogue threads (named barrier 1)
__device__ __forceinline__ bool epi_all(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, 1, 256, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t) v)
        : "memory");
    return r != 0;
}

// YT: TPMD_DTYPE_* of Y
template <int YT>
__global__ void __launch_bounds__(f8_cfg::THREADS, 1)
gemm_f8_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const f8_params p) {
    using cfg = f8_cfg;
    extern __shared__ uint8_t smem_raw[];
    __shared__ float red[2][cfg::BM];
    uint8_t *smem = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    uint64_t *bars = (uint64_t *) (smem + cfg::STAGES * cfg::STAGE_BYTES);
    uint32_t *tmem_slot = (uint32_t *) (bars + cfg::NBARS);
    auto A = [&](int s) { return smem_u32(smem) + s * cfg::STAGE_BYTES; };
    auto B = [&](int s) { return A(s) + cfg::A_BYTES; };
    auto full = [&](int s) { return smem_u32(&bars[s]); };
    auto empty = [&](int s) { return smem_u32(&bars[cfg::STAGES + s]); };
    auto tfull = [&](int a) { return smem_u32(&bars[2 * cfg::STAGES + a]); };
    auto tempty = [&](int a) { return smem_u32(&bars[2 * cfg::STAGES + cfg::NACC + a]); };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nb = blockIdx.x % p.tiles_n, n0 = nb * cfg::BN, m0 = (blockIdx.x / p.tiles_n) * cfg::BM;
    const int nk = p.kblocks;

    if (threadIdx.x == 0) {
        for (int s = 0; s < cfg::STAGES; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < cfg::NACC; a++) {
            mbar_init(tfull(a), 1);
            mbar_init(tempty(a), cfg::NEPI);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(cfg::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {  // TMA producer
            int issued = 0;
            for (int i = 0; i < nk; i++) {
                const int s = i % cfg::STAGES;
                if (i >= cfg::STAGES && !mbar_wait(empty(s), ((i / cfg::STAGES) - 1) & 1)) {
                    ok = false;
                    break;
                }
                mbar_expect_tx(full(s), cfg::STAGE_BYTES);
                tma_load_2d(A(s), &tmX, full(s), i * cfg::KB, m0);
                tma_load_2d(B(s), &tmW, full(s), i * cfg::KB, n0);
                issued++;
            }
            // the copies in flight land before the CTA goes on
            for (int j = issued > cfg::STAGES ? issued - cfg::STAGES : 0; j < issued; j++)
                if (!mbar_wait(full(j % cfg::STAGES), (j / cfg::STAGES) & 1)) ok = false;
            if (!ok) atomicExch(p.err, 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {  // MMA issuer
            int done = 0;
            for (int i = 0; i < nk; i++, done++) {
                const int s = i % cfg::STAGES, a = i % cfg::NACC;
                if (!mbar_wait(full(s), (i / cfg::STAGES) & 1) ||
                    (i >= cfg::NACC && !mbar_wait(tempty(a), ((i / cfg::NACC) - 1) & 1))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < cfg::KB / 32; kk++)
                    umma_f8(tmem + a * cfg::BN, smem_desc(A(s) + kk * 32, 1024, 2), smem_desc(B(s) + kk * 32, 1024, 2),
                            cfg::IDESC, kk > 0);
                umma_commit(empty(s));
                umma_commit(tfull(a));
            }
            // the MMAs in flight end before TMEM is freed
            for (int j = max(0, done - cfg::NACC); j < done; j++)
                if (!mbar_wait(tfull(j % cfg::NACC), (j / cfg::NACC) & 1)) ok = false;
            if (!ok) atomicExch(p.err, 1);
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2, row = q * 32 + lane, m = m0 + row;
        const uint32_t taddr = tmem + ((uint32_t) (q * 32) << 16) + half * 64;
        const float *sxr = p.sx + (int64_t) (m < p.M ? m : 0) * p.ldsx, *swr = p.sw + (int64_t) nb * p.ldsw;
        float acc[64];
#pragma unroll
        for (int c = 0; c < 64; c++) acc[c] = 0.0f;
        float sc = __ldg(sxr) * __ldg(swr);
        for (int i = 0; i < nk; i++) {
            const int a = i % cfg::NACC;
            const float next = i + 1 < nk ? __ldg(sxr + i + 1) * __ldg(swr + i + 1) : 0.0f;
            if (!mbar_wait(tfull(a), (i / cfg::NACC) & 1)) {
                ok = false;
                break;
            }
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t r[32];
                tmem_ld32(taddr + a * cfg::BN + c, r);
#pragma unroll
                for (int j = 0; j < 32; j++) acc[c + j] = fmaf(__uint_as_float(r[j]), sc, acc[c + j]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty(a));
            sc = next;
        }
        ok = epi_all(ok);
        if (!ok) {
            if (threadIdx.x == 64) atomicExch(p.err, 1);
        } else {
            const int n = n0 + half * 64;
#pragma unroll
            for (int c = 0; c < 64; c++)
                acc[c] = act_fn(acc[c] + (p.bias && n + c < p.N ? __ldg(p.bias + n + c) : 0.0f), p.act);
            if constexpr (YT == TPMD_DTYPE_F8) {
                float a = 0.0f;
#pragma unroll
                for (int c = 0; c < 64; c++)
                    if (n + c < p.N) a = fmaxf(a, fabsf(acc[c]));
                red[half][row] = a;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float s = fmaxf(__fdiv_rn(fmaxf(red[0][row], red[1][row]), F8_MAX), S_MIN);
                if (m < p.M) {
                    alignas(16) uint8_t v[64];
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        const uint16_t two = __nv_cvt_float2_to_fp8x2(
                            make_float2(__fdiv_rn(acc[c], s), __fdiv_rn(acc[c + 1], s)), __NV_SATFINITE, __NV_E4M3);
                        v[c] = (uint8_t) two;
                        v[c + 1] = (uint8_t) (two >> 8);
                    }
                    store_cols((uint8_t *) p.Y + (int64_t) m * p.ldy, v, n, p.N, p.y_vec);
                    if (half == 0) p.sy[(int64_t) m * p.ldsy + nb] = s;
                }
            } else if (m < p.M) {
                if constexpr (YT == TPMD_DTYPE_F16) {
                    alignas(16) __half v[64];
#pragma unroll
                    for (int c = 0; c < 64; c++) v[c] = __float2half_rn(acc[c]);
                    store_cols((__half *) p.Y + (int64_t) m * p.ldy, v, n, p.N, p.y_vec);
                } else {
                    store_cols((float *) p.Y + (int64_t) m * p.ldy, acc, n, p.N, p.y_vec);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cfg::TMEM_COLS)
                     : "memory");
}

bool encode_bytes(CUtensorMap *tm, const void *base, int64_t cols, int64_t rows, int64_t ld, int box_rows) {
    auto enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t) cols, (cuuint64_t) rows};
    const cuuint64_t strides[1] = {(cuuint64_t) ld};
    const cuuint32_t box[2] = {128, (cuuint32_t) box_rows}, estr[2] = {1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *) base, dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int YT>
cudaError_t run_f8(const CUtensorMap &tmX, const CUtensorMap &tmW, const f8_params &p, unsigned tiles,
                   cudaStream_t st) {
    static std::mutex mu;
    static uint64_t attr_set = 0;  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> g(mu);
        if (!(attr_set >> (dev & 63) & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(gemm_f8_kernel<YT>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, f8_cfg::SMEM);
            if (e != cudaSuccess) return e;
            attr_set |= 1ull << (dev & 63);
        }
    }
    gemm_f8_kernel<YT><<<tiles, f8_cfg::THREADS, f8_cfg::SMEM, st>>>(tmX, tmW, p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace tpmd

extern "C" int tpk_gemm_f8(const void *X, int64_t ldx, const float *sx, int64_t ldsx, const void *W, int64_t ldw,
                           const float *sw, int64_t ldsw, void *Y, int64_t ldy, int y_dtype, float *sy, int64_t ldsy,
                           int M, int N, int K, const float *bias, int act, void *stream) {
    using namespace tpmd;
    auto fail = [](const char *m) { return tpk_fail(std::string("tpk_gemm_f8: ") + m); };
    if (y_dtype != TPMD_DTYPE_F32 && y_dtype != TPMD_DTYPE_F16 && y_dtype != TPMD_DTYPE_F8) return fail("y_dtype");
    if (act < 0 || act > 3) return fail("act");
    if (M < 0 || N < 0 || K <= 0) return fail("bad shape");
    if ((y_dtype == TPMD_DTYPE_F8) != (sy != nullptr) && M > 0 && N > 0) return fail("sy goes with an F8 Y, and only with it");
    if (M == 0 || N == 0) return 0;
    if (!X || !sx || !W || !sw || !Y) return fail("null pointer");
    // a single row has no stride of its own
    if (M == 1) ldx = std::max<int64_t>(ldx, K) + 15 & ~(int64_t) 15;
    if (N == 1) ldw = std::max<int64_t>(ldw, K) + 15 & ~(int64_t) 15;
    if (((uintptr_t) X | (uintptr_t) W) & 15 || ldx % 16 || ldw % 16)
        return fail("X and W need 16-byte aligned bases and row strides");
    const int kblocks = (K + 127) / 128;
    if (ldx < K || ldw < K || ldx >= 1ll << 40 || ldw >= 1ll << 40 || (M > 1 && (ldy < N || ldsx < kblocks)) ||
        (N > 128 && ldsw < kblocks) || (sy && M > 1 && ldsy < (N + 127) / 128))
        return fail("bad row stride");
    if (((uintptr_t) sx | (uintptr_t) sw | (uintptr_t) sy | (uintptr_t) bias) & 3 ||
        (y_dtype != TPMD_DTYPE_F8 && (uintptr_t) Y & (y_dtype == TPMD_DTYPE_F16 ? 1 : 3)))
        return fail("a pointer is not aligned to its element type");
    const void *ptrs[] = {X, sx, W, sw, Y, sy, bias};
    tpk_device_scope dev(ptrs, 7);
    if (!dev.ok()) return fail(dev.why);
    f8_params p{};
    p.M = M;
    p.N = N;
    p.K = K;
    p.kblocks = kblocks;
    p.tiles_n = (N + 127) / 128;
    p.sx = sx;
    p.sw = sw;
    p.bias = bias;
    p.ldsx = ldsx;
    p.ldsw = ldsw;
    p.Y = Y;
    p.ldy = ldy;
    p.sy = sy;
    p.ldsy = ldsy;
    p.act = act;
    const int es = y_dtype == TPMD_DTYPE_F32 ? 4 : y_dtype == TPMD_DTYPE_F16 ? 2 : 1;
    p.y_vec = !((uintptr_t) Y & 15) && (M == 1 || ldy * es % 16 == 0);
    p.err = tpk_err_word();
    const int64_t tiles = (int64_t) p.tiles_n * ((M + 127) / 128);
    if (tiles > INT32_MAX) return fail("too many tiles");
    CUtensorMap tmX, tmW;
    if (!p.err || !encode_bytes(&tmX, X, K, M, ldx, 128) || !encode_bytes(&tmW, W, K, N, ldw, 128)) {
        cudaGetLastError();
        return fail("set-up failed");
    }
    cudaStream_t st = (cudaStream_t) stream;
    const cudaError_t e = y_dtype == TPMD_DTYPE_F32   ? run_f8<TPMD_DTYPE_F32>(tmX, tmW, p, (unsigned) tiles, st)
                          : y_dtype == TPMD_DTYPE_F16 ? run_f8<TPMD_DTYPE_F16>(tmX, tmW, p, (unsigned) tiles, st)
                                                      : run_f8<TPMD_DTYPE_F8>(tmX, tmW, p, (unsigned) tiles, st);
    if (e != cudaSuccess) return fail(cudaGetErrorString(e));
    return 0;
}
