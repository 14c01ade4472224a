// The product of two block-quantised 8-bit matrices on the tcgen05 tensor
// cores (tpk_gemm_f8, include/tpmd.h):
//
//   Y[m][n] = act( sum_b sx[m][b] sw[n/128][b] P_b[m][n] + bias[n] ),
//   P_b[m][n] = sum_{k in block b} X[m][k] W[n][k],  blocks of 128 along k
//
// An output tile is 128 x 128, or 256 x 256 of a pair of CTAs (cta_group::2:
// each loads 128 rows of X and 128 of W a k block, half of what it
// multiplies; a tile of its own would need more from L2 than the SMs get).
// Rows of X are the MMA's M side (TMEM lanes), blocks of 128 rows of W its N
// side, so a block's W scale of one k block is one number and a lane's
// factor sx sw is one number for all its 128 columns. Each k block of 128 is
// one pipeline stage (one 128-byte swizzled row a matrix row) and one MMA
// group into an accumulator of its own out of a ring in TMEM; the epilogue warps (each a lane quarter
// and half of the columns) read it, scale it and add it to f32 registers while the
// next blocks multiply. The products of e4m3 values are exact in
// f32; sums are f32 throughout.
//
// With 256 x 256 tiles (products that fill the SMs) CTAs are persistent: the
// loads and products of the next tile run on while a tile is written. With
// 128 x 128 tiles a CTA has one, and where SMs are left they have fewer rows
// or the k blocks of a tile are shared out over a cluster of up to eight CTAs; each leaves its
// partial tile in its shared memory, and each adds its rows of all of them
// (distributed shared memory), always in the same order.
//
// Measured, and what bounds it (f32 sums of every block of 128 pass through
// the epilogue warps):
//  * 8192 x 4096 x 4096, f16 out: 135 to 139 us, 2.0 PFLOP/s, 0.6 of twice the
//    bf16 rate (163 to 173 us after seconds under the power cap). The tensor
//    pipe is busy 48% of the time and no other pipe or memory more than a
//    third: the epilogue warps take a block in four rounds of read, wait for
//    the read, multiply-add, one after the other, and have a block's
//    accumulator till the last.
//  * 180 x 4096 x 1024 with tanh GELU and an 8-bit output: 8.6 us, 180 x 1024 x
//    4096: 8.5 us; by latency: launch, first loads, eight blocks, the join
//    (warps stall for instructions and loads, every pipe below 11%).
//  * 14 x 6656 x 4992 (33 MB of W): 11 us, 3.0 TB/s, 104 CTAs.
//  * 900 x 8192 x 453 with an 8-bit output: 15 us, with tanh GELU 28, with erf
//    GELU 35; two tiles for each pair of CTAs, their epilogues longer than
//    their products. (128 x 128 tiles instead: 34, 39, 45 us.)
//
// Every pipeline wait is bounded; an expired wait sets *err and the CTA
// skips the rest of its work.
#include <cuda_fp16.h>

#include "f8.cuh"
#include "tc_ops.cuh"
#include "tpmd_internal.h"
#include "../../include/tpmd.h"

#include <algorithm>
#include <cstring>
#include <mutex>
#include <string>

namespace tpmd {
namespace {

// NB = 2: of a pair of CTAs, issued by its first one
template <int NB>
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    const uint32_t mask = 0;
    if constexpr (NB == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(mask));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(mask));
}
// arrival on `bar` (NB = 2: of both CTAs) once the MMAs issued so far are done
template <int NB>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (NB == 1)
        umma_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t) 3)
            : "memory");
}
__device__ __forceinline__ uint32_t first_cta(uint32_t saddr) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(saddr));
    return a;
}
// a 128 x 128 tile; NB = 2: its bytes count on the first CTA's barrier
template <int NB>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int c0, int c1) {
    if constexpr (NB == 1)
        tma_load_2d(dst, tm, bar, c0, c1);
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
            "l"((uint64_t) tm), "r"(first_cta(bar)), "r"(c0), "r"(c1)
            : "memory");
}
// arrival on the first CTA's barrier, after reads of TMEM that a wait has
// ended: nothing in memory to publish, so no cluster-scope release (its memory
// barrier took over half of the warps' time here)
template <int NB>
__device__ __forceinline__ void arrive_first(uint32_t bar) {
    if constexpr (NB == 1)
        mbar_arrive(bar);
    else
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(first_cta(bar)) : "memory");
}
template <int NB>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    if constexpr (NB == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int NB>
__device__ __forceinline__ void tmem_dealloc(uint32_t tmem, uint32_t cols) {
    if constexpr (NB == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// of four values; erf by a call, so that the epilogues stay within the
// instruction caches
__device__ __noinline__ float4 gelu_erf4(float4 v) {
    constexpr float R = 0.70710678118654752f;
    return make_float4(0.5f * v.x * (1.0f + erff(v.x * R)), 0.5f * v.y * (1.0f + erff(v.y * R)),
                       0.5f * v.z * (1.0f + erff(v.z * R)), 0.5f * v.w * (1.0f + erff(v.w * R)));
}
// 0.5 v (1 + tanh u) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
__device__ __forceinline__ float gelu_tanh(float v) {
    return __fdividef(v, 1.0f + __expf(v * fmaf(-0.0713548162726f, v * v, -1.5957691216057308f)));
}
__device__ __forceinline__ float4 act4(float4 v, int act) {
    if (act == 1) return gelu_erf4(v);
    if (act == 2) return make_float4(gelu_tanh(v.x), gelu_tanh(v.y), gelu_tanh(v.z), gelu_tanh(v.w));
    if (act == 3)
        return make_float4(fmaxf(v.x, 0.2f * v.x), fmaxf(v.y, 0.2f * v.y), fmaxf(v.z, 0.2f * v.z), fmaxf(v.w, 0.2f * v.w));
    return v;
}

// NB: blocks of 128 columns a tile
template <int NB>
struct f8_cfg {
    // rows of a CTA; CTAs a tile (NB of them share an MMA: each holds 128 rows
    // of X and 128 of W, and the accumulators of its rows for all columns)
    static constexpr int BM = 128, BN = 128 * NB, KB = 128;
    static constexpr int A_BYTES = BM * KB, B_BYTES = 128 * KB, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = NB == 2 ? 5 : 6, NACC = 4 / NB;
    static constexpr uint32_t TMEM_COLS = 512;
    // D f32 (bit 4); A and B e4m3 (0 at bits 7 and 10); K-major both; N >> 3 at bit 17; M >> 4 at bit 24
    static constexpr uint32_t IDESC = (1u << 4) | ((uint32_t) (BN >> 3) << 17) | ((uint32_t) (BM * NB >> 4) << 24);
    static constexpr int CW = 64 * NB;  // columns an epilogue warp
    static constexpr int NEPI = 8, THREADS = 64 + 32 * NEPI;
    static constexpr int FR = 16;  // k blocks of factors kept
    static constexpr int NBARS = 2 * STAGES + 2 * NACC + FR;
    // NB = 2: a warp's staged 32 rows of 64 bytes; NB = 1: floats a row of a partial tile (16-byte bank shifts)
    static constexpr int PIECE = NB == 2 ? 32 * 64 : 0, PART_LD = 132;
    static constexpr int PIECE_BYTES = NEPI * PIECE;
    static constexpr int FACTORS = FR * (BM + NB);  // floats: sx of the rows, sw of the blocks
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + PIECE_BYTES + FACTORS * 4 + NBARS * 8 + 16;
    static_assert(FR >= STAGES + NACC, "factors outlive the products before them");
    static_assert(FACTORS % 2 == 0, "barrier alignment");
    static_assert(SMEM <= 232448, "shared memory");
    static_assert(BM * PART_LD * 4 <= STAGES * STAGE_BYTES, "a partial tile fits the stages");
};

struct f8_params {
    int M, N, K, kblocks, tiles_n, tiles, splits, kb_per_split;
    int bm;            // NB = 1: rows from a tile to the next
    uint32_t x_bytes;  // of X a stage
    const float *sx, *sw, *bias;
    int64_t ldsx, ldsw;
    void *Y;
    int64_t ldy;
    float *sy;
    int64_t ldsy;
    int act;
    bool w_pre;  // W's first tiles load before the programmatic-dependence wait
    bool y_vec;  // Y takes stores of four elements (NB = 2: of 16 bytes)
    int *err;
};

// (a0, a1) += (x0, x1) * s, two f32 multiply-adds in one instruction
__device__ __forceinline__ void fma2(float &a0, float &a1, uint32_t x0, uint32_t x1, float s) {
    asm("{\n\t.reg .b64 a, x, f;\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mov.b64 f, {%4, %4};\n\t"
        "fma.rn.f32x2 a, x, f, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "r"(x0), "r"(x1), "f"(s));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float4 ld_rank4(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
// 32 rows of 64 staged bytes (below: unit u of row r at u ^ (r / 2 mod 4)) to
// `rows` rows of Y, `cols` columns of ES bytes, where rows start off 16-byte
// boundaries or end: an element a lane, one behind the other
template <int ES>
__device__ __noinline__ void copy_elements(uint8_t *y, int64_t step, const uint8_t *piece, int rows, int cols, int lane) {
    constexpr int PER = 64 / ES;  // elements a row
#pragma unroll 4
    for (int i = lane; i < 32 * PER; i += 32) {
        const int r = i / PER, c = i % PER, at = c * ES;
        const uint8_t *x = piece + r * 64 + (at / 16 ^ (r >> 1 & 3)) * 16 + at % 16;
        if (r < rows && c < cols) {
            if (ES == 4) *reinterpret_cast<uint32_t *>(y + r * step + at) = *reinterpret_cast<const uint32_t *>(x);
            else if (ES == 2) *reinterpret_cast<uint16_t *>(y + r * step + at) = *reinterpret_cast<const uint16_t *>(x);
            else y[r * step + at] = *x;
        }
    }
}
// a row of 128 columns, four a lane, to Y where it starts off a vector's
// boundary or ends (F8: quantised by s): through `row` in shared memory, so
// that lanes store one behind the other
template <int YT>
__device__ __noinline__ void store_off(const f8_params &p, int64_t m, int n0, float4 v, f8_scale s, float *row, int lane) {
    if constexpr (YT == TPMD_DTYPE_F8) reinterpret_cast<uint32_t *>(row)[lane] = f8_quant4(v.x, v.y, v.z, v.w, s);
    else reinterpret_cast<float4 *>(row)[lane] = v;
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int c = lane + 32 * e;
        if (n0 + c < p.N) {
            const int64_t at = m * p.ldy + n0 + c;
            if constexpr (YT == TPMD_DTYPE_F8) ((uint8_t *) p.Y)[at] = reinterpret_cast<const uint8_t *>(row)[c];
            else if constexpr (YT == TPMD_DTYPE_F16) ((__half *) p.Y)[at] = __float2half_rn(row[c]);
            else ((float *) p.Y)[at] = row[c];
        }
    }
}

// YT: TPMD_DTYPE_* of Y
template <int YT, int NB>
__global__ void __launch_bounds__(f8_cfg<NB>::THREADS, 1)
gemm_f8_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
               const __grid_constant__ f8_params p) {
    using cfg = f8_cfg<NB>;
    constexpr int ST = cfg::STAGES, NA = cfg::NACC, ES = YT == TPMD_DTYPE_F32 ? 4 : YT == TPMD_DTYPE_F16 ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    uint8_t *pieces = smem + ST * cfg::STAGE_BYTES;
    float *fsx = (float *) (pieces + cfg::PIECE_BYTES), *fsw = fsx + cfg::FR * cfg::BM;  // [FR][BM], [FR][NB]
    uint64_t *bars = (uint64_t *) (fsx + cfg::FACTORS);
    uint32_t *tmem_slot = (uint32_t *) (bars + cfg::NBARS);
    auto A = [&](int s) { return smem_u32(smem) + s * cfg::STAGE_BYTES; };
    auto B = [&](int s) { return A(s) + cfg::A_BYTES; };
    auto full = [&](int s) { return smem_u32(&bars[s]); };
    auto empty = [&](int s) { return smem_u32(&bars[ST + s]); };
    auto tfull = [&](int a) { return smem_u32(&bars[2 * ST + a]); };
    auto tempty = [&](int a) { return smem_u32(&bars[2 * ST + NA + a]); };
    auto ffull = [&](int i) { return smem_u32(&bars[2 * ST + 2 * NA + i]); };

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = NB == 2 ? blockIdx.x % 2 : 0;  // of the CTA pair (its even CTA issues the MMAs)
    const int split = NB == 1 ? blockIdx.x % p.splits : 0;
    const int cta = NB == 1 ? blockIdx.x / p.splits : blockIdx.x / 2, ctas = NB == 1 ? gridDim.x / p.splits : gridDim.x / 2;
    const int kb0 = split * p.kb_per_split, nk = min(p.kblocks - kb0, p.kb_per_split);  // nk >= 1 (host)

    if (threadIdx.x == 32) {
        prefetch_map(&tmX);
        prefetch_map(&tmW);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < NA; a++) {
            mbar_init(tfull(a), 1);
            mbar_init(tempty(a), cfg::NEPI * NB);
        }
        for (int i = 0; i < cfg::FR; i++) mbar_init(ffull(i), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<NB>(smem_u32(tmem_slot), cfg::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    if (NB == 2) cluster_sync();  // the pair's barriers are set up
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        // TMA producer, and the factors of each k block into their ring: four
        // rows' sx a lane, loaded four blocks ahead. Block c's slot was last read
        // for block c - FR, and its stage is free only when the products of
        // block c - ST are done, which began after block c - ST - NA was read.
        // (a programmatic dependent starts while the kernel before it runs: all
        // that this one reads of it, and writes, comes after this wait)
        // (but W, where that kernel does not write it)
        const int pre = NB == 1 && p.w_pre ? min(nk, ST) : 0;
        if (pre && elect_one())
            for (int i = 0; i < pre; i++) {
                mbar_expect_tx(full(i), p.x_bytes + cfg::B_BYTES);
                load_tile<NB>(B(i), &tmW, full(i), (kb0 + i) * cfg::KB, cta % p.tiles_n * cfg::BN);
            }
        __syncwarp();
        pdl_wait();
        pdl_trigger();
        int c = 0;
        for (int tile = cta; ok && tile < p.tiles; tile += ctas) {
            const int n0 = tile % p.tiles_n * cfg::BN, m0 = (tile / p.tiles_n * NB + rank) * (NB == 2 ? 128 : p.bm);
            // (rows and blocks behind the last one have factors of the last one)
            const float *sx[4], *sw = p.sw + (int64_t) min(n0 / 128 + lane % NB, (p.N - 1) / 128) * p.ldsw + kb0;
#pragma unroll
            for (int r = 0; r < 4; r++) sx[r] = p.sx + (int64_t) min(m0 + lane + 32 * r, p.M - 1) * p.ldsx + kb0;
            float x[4][4], w[4], nx[4][4], nw[4];  // of four blocks, and of the four after them
            auto fetch = [&](int i0) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = min(i0 + e, nk - 1);
                    nw[e] = sw[i];
#pragma unroll
                    for (int r = 0; r < 4; r++) nx[e][r] = sx[r][i];
                }
            };
            fetch(0);
            for (int i0 = 0; ok && i0 < nk; i0 += 4) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[e] = nw[e];
#pragma unroll
                    for (int r = 0; r < 4; r++) x[e][r] = nx[e][r];
                }
                if (i0 + 4 < nk) fetch(i0 + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (i0 + e >= nk) break;
                    const int s = c % ST, f = c % cfg::FR;
                    if (c >= ST && !warp_wait(empty(s), ((c / ST) - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        // the bytes of both CTAs of a pair count on its first one's barrier
                        if (rank == 0 && c >= pre) mbar_expect_tx(full(s), (p.x_bytes + cfg::B_BYTES) * NB);
                        load_tile<NB>(A(s), &tmX, full(s), (kb0 + i0 + e) * cfg::KB, m0);
                        if (c >= pre) load_tile<NB>(B(s), &tmW, full(s), (kb0 + i0 + e) * cfg::KB, n0 + rank * 128);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) fsx[f * cfg::BM + lane + 32 * r] = x[e][r];
                    if (lane < NB) fsw[f * NB + lane] = w[e];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(ffull(f));
                    c++;
                }
            }
        }
        // the copies in flight land (and are read) before the CTA goes on
        for (int j = max(0, c - ST); j < c; j++)
            if (!warp_wait(empty(j % ST), (j / ST) & 1)) ok = false;
        if (!ok && lane == 0) atomicExch(p.err, 1);
    } else if (warp == 1) {
        if (rank == 0) {
            // MMA issuer: the whole warp goes through the loop, so that what it
            // computes stays in uniform registers, and one lane issues (a loop of
            // one lane alone took longer to issue the MMAs than they run)
            int c = 0;
            for (int tile = cta; ok && tile < p.tiles; tile += ctas)
                for (int i = 0; i < nk; i++, c++) {
                    const int s = c % ST, a = c % NA;
                    ok = c < NA ? warp_wait(full(s), (c / ST) & 1)
                                : warp_wait2(full(s), (c / ST) & 1, tempty(a), ((c / NA) - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t ad = smem_desc(A(s), 1024, 2), bd = smem_desc(B(s), 1024, 2);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < cfg::KB / 32; kk++)
                            umma_f8<NB>(tmem + a * cfg::BN, ad + kk * 2, bd + kk * 2, cfg::IDESC, kk > 0);
                        commit<NB>(tfull(a));
                        commit<NB>(empty(s));
                    }
                    __syncwarp();
                }
            // the MMAs in flight end before TMEM is freed
            for (int j = max(0, c - NA); j < c; j++)
                if (!warp_wait(tfull(j % NA), (j / NA) & 1)) ok = false;
            if (!ok && lane == 0) atomicExch(p.err, 1);
        }
    } else {
        // a warp: a lane quarter (32 rows) and half of the columns (half a block
        // of 128, or one of two)
        constexpr int CW = cfg::CW;
        const int q = warp & 3, half = (warp - 2) >> 2, blk = half * CW / 128;
        const uint32_t taddr = tmem + ((uint32_t) (q * 32) << 16) + half * CW;
        uint8_t *piece = pieces + (warp - 2) * cfg::PIECE;
        int c = 0;
        for (int tile = cta; ok && tile < p.tiles; tile += ctas) {
            const int n0 = tile % p.tiles_n * cfg::BN + half * CW, nb = n0 / 128;
            const int m0 = (tile / p.tiles_n * NB + rank) * (NB == 2 ? 128 : p.bm) + q * 32;
            float acc[CW];
#pragma unroll
            for (int e = 0; e < CW; e++) acc[e] = 0.0f;
            // four blocks' factors at a time, once the last of them is there (the
            // TMA warp is that far ahead: the fifth block after the one being
            // read waits for the products of that one only)
            static_assert(ST >= 4, "the TMA warp may run four blocks ahead");
            float f4[4];
            for (int i = 0; i < nk; i++, c++) {
                const int a = c % NA;
                if (i % 4 == 0) {
                    const int last = c + min(3, nk - 1 - i);
                    ok = warp_wait2(ffull(last % cfg::FR), (last / cfg::FR) & 1, tfull(a), (c / NA) & 1);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int f = min(c + e, last) % cfg::FR;
                        f4[e] = fsx[f * cfg::BM + q * 32 + lane] * fsw[f * NB + blk];
                    }
                } else {
                    ok = warp_wait(tfull(a), (c / NA) & 1);
                }
                if (!ok) break;
                const float scale = i % 4 == 0 ? f4[0] : i % 4 == 1 ? f4[1] : i % 4 == 2 ? f4[2] : f4[3];
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < CW; x += 32) {
                    uint32_t r[32];
                    tmem_ld32(taddr + a * cfg::BN + x, r);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) fma2(acc[x + j], acc[x + j + 1], r[j], r[j + 1], scale);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_first<NB>(tempty(a));
            }
            if (NB == 1) {  // the (partial) tile into the stages (one tile a CTA, its products are in)
                if (!ok) break;
#pragma unroll
                for (int e = 0; e < CW; e += 4)
                    *reinterpret_cast<float4 *>((float *) smem + (q * 32 + lane) * cfg::PART_LD + half * CW + e) =
                        make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                break;
            }
            if constexpr (NB == 2) {
                if (!ok) break;
                // bias and activation in place (the same columns in every lane;
                // one test of the activation, not one for every four columns)
                if (p.bias) {
#pragma unroll
                    for (int e = 0; e < CW; e++) acc[e] += p.bias[min(n0 + e, p.N - 1)];
                }
                auto activate = [&](auto f) {
#pragma unroll
                    for (int e = 0; e < CW; e += 4) {
                        const float4 v = f(make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]));
                        acc[e] = v.x;
                        acc[e + 1] = v.y;
                        acc[e + 2] = v.z;
                        acc[e + 3] = v.w;
                    }
                };
                if (p.act == 1) activate([](float4 v) { return gelu_erf4(v); });
                else if (p.act == 2) activate([](float4 v) { return act4(v, 2); });
                else if (p.act == 3) activate([](float4 v) { return act4(v, 3); });
                f8_scale k = {1.0f, 1.0f};
                if constexpr (YT == TPMD_DTYPE_F8) {
                    float top = 0.0f;
                    // (columns behind the last one hold act(its bias); a test a
                    // column took 5% of 8192 x 4096 x 1024, so only here)
                    if (n0 + CW <= p.N) {
#pragma unroll
                        for (int e = 0; e < CW; e++) top = fmaxf(top, fabsf(acc[e]));
                    } else {
#pragma unroll
                        for (int e = 0; e < CW; e++)
                            if (n0 + e < p.N) top = fmaxf(top, fabsf(acc[e]));
                    }
                    k = f8_scale_of(top);
                    if (m0 + lane < p.M && n0 < p.N) p.sy[(int64_t) (m0 + lane) * p.ldsy + nb] = k.s;
                }
                // 64 bytes of each row at a time through shared memory, 16-byte
                // unit u of row r at u ^ (r / 2 mod 4) against bank conflicts:
                // a store covers eight rows
                constexpr int PER = 16 / ES;
                const int sub = lane / 4, unit = lane % 4;
                uint8_t *y = (uint8_t *) p.Y + ((int64_t) (m0 + sub) * p.ldy + n0 + unit * PER) * ES;
                const int64_t step = 8 * p.ldy * ES;
                const uint8_t *src = piece + sub * 64 + (unit ^ (sub >> 1 & 3)) * 16;  // (row + 8: the same unit)
                uint8_t *own = piece + lane * 64;
                const bool whole = p.y_vec && n0 + CW <= p.N;
                const int rows_left = p.M - m0 - sub;
#pragma unroll
                for (int x = 0; x < CW; x += 4 * PER) {
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        uint4 w;
                        const float *v = acc + x + u * PER;
                        if constexpr (YT == TPMD_DTYPE_F32) {
                            w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                           __float_as_uint(v[3]));
                        } else if constexpr (YT == TPMD_DTYPE_F16) {
                            const __half2 h[4] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3]),
                                                  __floats2half2_rn(v[4], v[5]), __floats2half2_rn(v[6], v[7])};
                            w = *reinterpret_cast<const uint4 *>(h);
                        } else {
                            w = make_uint4(f8_quant4(v[0], v[1], v[2], v[3], k), f8_quant4(v[4], v[5], v[6], v[7], k),
                                           f8_quant4(v[8], v[9], v[10], v[11], k),
                                           f8_quant4(v[12], v[13], v[14], v[15], k));
                        }
                        *reinterpret_cast<uint4 *>(own + (u ^ (lane >> 1 & 3)) * 16) = w;
                    }
                    __syncwarp();
                    if (whole) {
                        uint4 t[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) t[r] = *reinterpret_cast<const uint4 *>(src + r * 512);
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (r * 8 < rows_left) *reinterpret_cast<uint4 *>(y + r * step + x * ES) = t[r];
                    } else {
                        copy_elements<ES>((uint8_t *) p.Y + ((int64_t) m0 * p.ldy + n0 + x) * ES, p.ldy * ES, piece,
                                          p.M - m0, p.N - n0 - x, lane);
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok && lane == 0) atomicExch(p.err, 1);
    }
    if (NB == 1) {
        // each CTA of the cluster adds its share of the rows over all
        // splits (always in the same order), a warp a row
        __syncwarp();
        if (p.splits > 1) cluster_sync();
        else __syncthreads();
        const int n0 = cta % p.tiles_n * 128, m0 = cta / p.tiles_n * p.bm, n = n0 + lane * 4;
        const uint32_t part = smem_u32(smem) + lane * 16;
        float bias[4];
#pragma unroll
        for (int e = 0; e < 4; e++) bias[e] = p.bias && n + e < p.N ? p.bias[n + e] : 0.0f;
        // four rows a warp at a time, three other CTAs' loads in flight together.
        // (Columns behind the last one are zeros or NaN: they do not count in a
        // row's maximum.)
        constexpr int RB = 4, NW = cfg::THREADS / 32;
        const int rows = min(p.bm, p.M - m0);
        const bool vec4 = p.y_vec && (n0 + 128 <= p.N || p.N % 4 == 0);
#pragma unroll 1
        for (int r0 = (split * NW + warp) * RB; r0 < rows; r0 += p.splits * NW * RB) {
            float4 v[RB];
#pragma unroll
            for (int j = 0; j < RB; j++) {
                v[j] = *reinterpret_cast<const float4 *>((const float *) smem + (r0 + j) * cfg::PART_LD + lane * 4);
                v[j] = make_float4(v[j].x + bias[0], v[j].y + bias[1], v[j].z + bias[2], v[j].w + bias[3]);
            }
#pragma unroll 1
            for (int k0 = 1; k0 < p.splits; k0 += 3) {
                float4 f[3][RB];
#pragma unroll
                for (int k = 0; k < 3; k++) {
                    // every CTA starts with the one after it: no two read one CTA's at a time
                    int from = split + k0 + k;
                    if (from >= p.splits) from -= p.splits;
#pragma unroll
                    for (int j = 0; j < RB; j++)
                        if (k0 + k < p.splits) f[k][j] = ld_rank4(part + (r0 + j) * cfg::PART_LD * 4, from);
                }
#pragma unroll
                for (int k = 0; k < 3; k++)
#pragma unroll
                    for (int j = 0; j < RB; j++)
                        if (k0 + k < p.splits) {
                            v[j].x += f[k][j].x;
                            v[j].y += f[k][j].y;
                            v[j].z += f[k][j].z;
                            v[j].w += f[k][j].w;
                        }
            }
            if (p.act == 2) {
#pragma unroll
                for (int j = 0; j < RB; j++) v[j] = act4(v[j], 2);
            } else if (p.act) {
#pragma unroll
                for (int j = 0; j < RB; j++) v[j] = act4(v[j], p.act);
            }
            float top[RB];
            if constexpr (YT == TPMD_DTYPE_F8) {
#pragma unroll
                for (int j = 0; j < RB; j++)
                    top[j] = fmaxf(fmaxf(fabsf(v[j].x), fabsf(v[j].y)), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
#pragma unroll
                for (int w = 16; w > 0; w >>= 1)
#pragma unroll
                    for (int j = 0; j < RB; j++) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], w));
            }
            const int64_t m = m0 + r0;
            uint8_t *y = (uint8_t *) p.Y + (m * p.ldy + n) * ES;
            const int64_t step = p.ldy * ES;
#pragma unroll
            for (int j = 0; j < RB; j++) {
                if (r0 + j >= rows) break;
                f8_scale s = {1.0f, 1.0f};
                if constexpr (YT == TPMD_DTYPE_F8) {
                    s = f8_scale_of(top[j]);
                    if (lane == 0) p.sy[(m + j) * p.ldsy + n0 / 128] = s.s;
                }
                if (!vec4) {
                    // (the row's place here: no other warp reads it)
                    store_off<YT>(p, m + j, n0, v[j], s, (float *) smem + (r0 + j) * cfg::PART_LD, lane);
                } else if (n < p.N) {
                    if constexpr (YT == TPMD_DTYPE_F8) {
                        *reinterpret_cast<uint32_t *>(y + j * step) = f8_quant4(v[j].x, v[j].y, v[j].z, v[j].w, s);
                    } else if constexpr (YT == TPMD_DTYPE_F16) {
                        const __half2 h[2] = {__floats2half2_rn(v[j].x, v[j].y), __floats2half2_rn(v[j].z, v[j].w)};
                        *reinterpret_cast<uint2 *>(y + j * step) = *reinterpret_cast<const uint2 *>(h);
                    } else {
                        *reinterpret_cast<float4 *>(y + j * step) = v[j];
                    }
                }
            }
        }
        if (p.splits > 1) cluster_sync();  // no CTA leaves while others read its partial
    }
    tc_fence_before();
    __syncthreads();
    if (NB == 2) cluster_sync();  // no CTA leaves while its pair uses its memory
    if (warp == 1) tmem_dealloc<NB>(tmem, cfg::TMEM_COLS);
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

template <int YT, int NB>
cudaError_t run_f8(const CUtensorMap &tmX, const CUtensorMap &tmW, const f8_params &p, cudaStream_t st) {
    using cfg = f8_cfg<NB>;
    static std::mutex mu;
    static uint64_t attr_set = 0;  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> g(mu);
        if (!(attr_set >> (dev & 63) & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(gemm_f8_kernel<YT, NB>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, cfg::SMEM);
            if (e != cudaSuccess) return e;
            attr_set |= 1ull << (dev & 63);
        }
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned) (NB == 1 ? p.tiles * p.splits : 2 * std::min(p.tiles, sm_count() / 2)), 1, 1);
    lc.blockDim = dim3(cfg::THREADS, 1, 1);
    lc.dynamicSmemBytes = cfg::SMEM;
    lc.stream = st;
    cudaLaunchAttribute at[2];
    int na = 0;
    if (NB == 2 || p.splits > 1) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim.x = (unsigned) (NB == 1 ? p.splits : 2);
        at[na].val.clusterDim.y = 1;
        at[na].val.clusterDim.z = 1;
        na++;
    }
    at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[na].val.programmaticStreamSerializationAllowed = 1;
    na++;
    lc.attrs = at;
    lc.numAttrs = na;
    const cudaError_t e = cudaLaunchKernelEx(&lc, gemm_f8_kernel<YT, NB>, tmX, tmW, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}
template <int YT>
cudaError_t run_f8(int nb, const CUtensorMap &tmX, const CUtensorMap &tmW, const f8_params &p, cudaStream_t st) {
    return nb == 2 ? run_f8<YT, 2>(tmX, tmW, p, st) : run_f8<YT, 1>(tmX, tmW, p, st);
}

}  // namespace

cudaError_t gemm_f8(const gemm_f8_desc &d, cudaStream_t st) {
    f8_params p{};
    const int kblocks = (d.K + 127) / 128;
    p.M = d.M;
    p.N = d.N;
    p.K = d.K;
    p.kblocks = kblocks;
    p.sx = d.sx;
    p.sw = d.sw;
    p.bias = d.bias;
    p.ldsx = d.ldsx;
    p.ldsw = d.ldsw;
    p.Y = d.Y;
    p.ldy = d.ldy;
    p.sy = d.sy;
    p.ldsy = d.ldsy;
    p.act = d.act;
    p.w_pre = d.w_const;
    p.err = d.err ? d.err : tpk_err_word();
    if (!p.err) return cudaErrorUnknown;
    const int es = d.y_dtype == TPMD_DTYPE_F32 ? 4 : d.y_dtype == TPMD_DTYPE_F16 ? 2 : 1;
    const int64_t nblk = (d.N + 127) / 128;
    // 256 x 256 tiles of CTA pairs where they fill the SMs; else 128 x 128
    const int nb = ((int64_t) d.M + 255) / 256 * ((nblk + 1) / 2) >= sm_count() / 2 ? 2 : 1;
    const int unit = nb == 2 ? 16 : 4 * es;
    p.y_vec = !((uintptr_t) d.Y & (unit - 1)) && (d.M == 1 || d.ldy * es % unit == 0);
    // 128 x 128: clusters that leave a CTA eight blocks; then, where SMs are
    // left, tiles of fewer rows (32 at least): W is read again from L2, but more
    // CTAs form the outputs. Few tiles all the same: clusters down to two
    // blocks. (Clusters down to two blocks alone, so: 1430 x 379 x
    // 181 12.5, 7.1 us; 777 x 1000 x 528 9.1, 8.0; 180 x 1024 x 1024 6.8, 6.3.
    // Fewer rows under clusters of four: 180 x 1024 x 4096 8.7 -> 9.3. Eight
    // blocks alone: 30 x 300 x 1500 6.0 -> 7.0.)
    p.tiles_n = (int) ((nblk + nb - 1) / nb);
    int64_t mtiles = ((int64_t) d.M + nb * 128 - 1) / (nb * 128);
    int splits = 1;
    if (nb == 1) {
        splits = cluster_size(mtiles * p.tiles_n, kblocks / 8);
        if (splits <= 2)
            mtiles = std::max(mtiles, std::min<int64_t>(sm_count() / splits / p.tiles_n, ((int64_t) d.M + 31) / 32));
        if (mtiles * p.tiles_n <= 16) splits = std::max(splits, cluster_size(mtiles * p.tiles_n, kblocks / 2));
    }
    // the tiles share the rows out evenly, and no box reaches far behind the
    // last row: its zeros take as long to write as data. (What the rest of a
    // tile's rows hold reaches no output. 14 x 6656 x 4992: 16.9 -> 11.1 us)
    p.bm = nb == 2 ? 128 : (int) ((d.M + mtiles - 1) / mtiles + 7) & ~7;
    p.x_bytes = p.bm * 128;
    if (nb == 1) mtiles = ((int64_t) d.M + p.bm - 1) / p.bm;
    if (mtiles * p.tiles_n > INT32_MAX / 8) return cudaErrorInvalidValue;
    p.tiles = (int) (mtiles * p.tiles_n);
    p.kb_per_split = (kblocks + splits - 1) / splits;
    p.splits = (kblocks + p.kb_per_split - 1) / p.kb_per_split;  // no empty split
    CUtensorMap tmX, tmW;
    if (!encode_bytes(&tmX, d.X, d.K, d.M, d.ldx, p.bm) || !encode_bytes(&tmW, d.W, d.K, d.N, d.ldw, 128))
        return cudaErrorInvalidValue;
    return d.y_dtype == TPMD_DTYPE_F32   ? run_f8<TPMD_DTYPE_F32>(nb, tmX, tmW, p, st)
           : d.y_dtype == TPMD_DTYPE_F16 ? run_f8<TPMD_DTYPE_F16>(nb, tmX, tmW, p, st)
                                         : run_f8<TPMD_DTYPE_F8>(nb, tmX, tmW, p, st);
}

}  // namespace tpmd

extern "C" int tpk_gemm_f8(const void *X, int64_t ldx, const float *sx, int64_t ldsx, const void *W, int64_t ldw,
                           const float *sw, int64_t ldsw, void *Y, int64_t ldy, int y_dtype, float *sy, int64_t ldsy,
                           int M, int N, int K, const float *bias, int act, void *stream) {
    using namespace tpmd;
    auto fail = [](const char *m) { return tpk_fail(std::string("tpk_gemm_f8: ") + m); };
    if (y_dtype != TPMD_DTYPE_F32 && y_dtype != TPMD_DTYPE_F16 && y_dtype != TPMD_DTYPE_F8) return fail("y_dtype");
    if (act < 0 || act > 3) return fail("act");
    if (M < 0 || N < 0 || K <= 0 || M > 1 << 30 || N > 1 << 30 || K > 1 << 30) return fail("bad shape");
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
    gemm_f8_desc d;
    d.X = X;
    d.ldx = ldx;
    d.sx = sx;
    d.ldsx = ldsx;
    d.W = W;
    d.ldw = ldw;
    d.sw = sw;
    d.ldsw = ldsw;
    d.Y = Y;
    d.ldy = ldy;
    d.y_dtype = y_dtype;
    d.sy = sy;
    d.ldsy = ldsy;
    d.M = M;
    d.N = N;
    d.K = K;
    d.bias = bias;
    d.act = act;
    const cudaError_t e = gemm_f8(d, (cudaStream_t) stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(e == cudaErrorInvalidValue ? "too many tiles, or the launch was refused" : cudaGetErrorString(e));
    }
    return 0;
}

extern "C" int tpk_gemm_f8_packed(const int64_t args[19]) {
    tpmd::packed_args p{args};
    const void *X = p.ptr();
    const int64_t ldx = p.i64();
    const float *sx = (const float *) p.ptr();
    const int64_t ldsx = p.i64();
    const void *W = p.ptr();
    const int64_t ldw = p.i64();
    const float *sw = (const float *) p.ptr();
    const int64_t ldsw = p.i64();
    void *Y = p.ptr();
    const int64_t ldy = p.i64();
    const int y_dtype = p.i32();
    float *sy = (float *) p.ptr();
    const int64_t ldsy = p.i64();
    const int M = p.i32(), N = p.i32(), K = p.i32();
    const float *bias = (const float *) p.ptr();
    const int act = p.i32();
    void *stream = p.ptr();
    if (!p.fits) return tpmd::tpk_fail("tpk_gemm_f8: an argument is out of its range");
    return tpk_gemm_f8(X, ldx, sx, ldsx, W, ldw, sw, ldsw, Y, ldy, y_dtype, sy, ldsy, M, N, K, bias, act, stream);
}
