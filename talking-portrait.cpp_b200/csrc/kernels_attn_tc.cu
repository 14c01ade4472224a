// Sliding-window attention with first tokens that stay visible
// (tpk_attn_window, include/tpmd.h) on the tcgen05 tensor cores, for f16:
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i),
//   over keys j < min(L, p + right + 1) with j >= p - left or j < sinks
//
// in one pass over the keys with a running maximum m and sum. Rows of the
// MMA are (token, query head of the group) pairs, so the query heads that
// share a key head read its keys once and a tile spans few positions. Keys
// come in tiles of 64: those of the window from its first key on (TMA boxes
// start at any row), then those of the sinks; the last tile of each is cut to
// a multiple of 16 keys.
//
// Per tile S = Q K^T (f32, TMEM), a thread per row turns S into weights P
// (f16, over S in TMEM), O += P V (f32, TMEM). The maximum that P is relative
// to moves only when a row's maximum has grown by 2^8, and O needs no
// rescaling until then. P holds 2^7 for the weight of that maximum, so up to
// 2^15: above, f16 ends at 2^16; below, weights keep 11 bits down to 2^-21 of
// it, and are off by 2^-32 of it at most under that. (With 1 for that weight,
// keys that weigh 2^-25 of it were lost to O and not to the sum: 2500 tokens
// of one large score and 2000 small ones came out as zeros. The matrix
// instruction takes no f32; P in two f16 parts would double half its work.)
//
// Two softmax warpgroups, each with an MMA warp of its own (the prompt below
// 495 -> 452 us; MMAs issued by one lane in a loop of its own, in place of a
// converged warp's elected lane, took 85 clocks each) and two buffers for S,
// so that the scores of the next tile are multiplied while a tile's weights
// are formed:
//  * prompts: each has its own 128 rows, both go through the same key tiles;
//  * few rows (SPLIT): both have the same rows and take alternate key tiles;
//    rows that fill no more than half or a quarter of the MMA's lanes are
//    loaded two or four times, and each copy's warps take that share of
//    every tile's keys; and the tiles are shared out over a cluster of up to
//    eight CTAs. Their parts (m, sum, O) join in shared memory, then over the
//    cluster (distributed shared memory), always in the same order.
//
// A weight of zero times a value that is not finite is NaN: the values of
// keys that no row of the CTA sees are cleared in shared memory, and a row
// that still comes out not finite is computed again on the CUDA cores from
// its visible keys alone.
//
// Measured, and what bounds it:
//  * 16384 tokens, 16 heads of 128 on 4, 4096 keys each (481 GFLOP): 451 us,
//    1.07 PFLOP/s, 0.63 of the matrix rate (524 us after seconds under the
//    power cap). The tensor pipe and the special-function pipe (all the
//    exponentials) are each busy half of the time: neither hides the other
//    wholly, nor the hand-over between them.
//  * 16 sequences of one token over 4100 keys, 16 heads of 128 on 4 (134 MB):
//    28 to 30 us, 4.5 to 4.8 TB/s, 0.7 of the copy rate: 128 CTAs, 20 SMs
//    without one, each ending with a join over its cluster.
//  * 7500 tokens, 12 heads of 64, 251 keys each: 31 us (360 CTAs in 2.4 waves
//    of up to nine tiles; tensor pipe 13%, special functions 27%: a CTA's
//    start and end, which nothing overlaps).
//
// Every pipeline wait is bounded; an expired wait sets *err and the CTA
// skips the rest of its work.
#include <cuda_fp16.h>

#include "attn_row.cuh"
#include "tc_ops.cuh"
#include "tpmd_internal.h"

#include <algorithm>
#include <mutex>

namespace tpmd {
namespace {

template <int DB, bool SPLIT>
struct at_cfg {
    static constexpr int KT = 64;                        // keys a tile
    static constexpr int Q_BYTES = 128 * 128 * DB;       // 128 rows of DB 64-column boxes
    static constexpr int TILE_BYTES = KT * 128 * DB;
    static constexpr int STAGE_BYTES = 2 * TILE_BYTES;   // a tile's V and a later one's K
    static constexpr int NQ = SPLIT ? 1 : 2;
    static constexpr int STAGES = DB == 2 ? (SPLIT ? 6 : 5) : 8;
    static constexpr int THREADS = 352;                  // 8 softmax warps, TMA, an MMA warp for each warpgroup
    static constexpr int OLD = DB * 64 + 4;              // floats a row of the joined parts (bank shift)
    static constexpr int NBARS = 2 * STAGES + 4 + 4 + 4 + 4;
    static constexpr int DATA = NQ * Q_BYTES + STAGES * STAGE_BYTES;
    static constexpr int SMEM = 1024 + DATA + NBARS * 8 + 16;
    static_assert(SMEM <= 232448, "shared memory");
    static_assert(!SPLIT || 256 * OLD * 4 <= STAGES * STAGE_BYTES, "parts fit the stages");
};
constexpr uint32_t TMEM_COLS = 512;
constexpr float P_EXP = 7.0f;  // P is 2^P_EXP at the maximum it is relative to

struct at_params {
    attn_desc d;
    int g, tb, reps, qtiles, splits;
    float c;  // scale log2(e)
    bool o_vec;
    int *err;
};

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int c0, int c1, int c2,
                                            int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"((uint64_t) tm), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}
// A in TMEM
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    const uint32_t mask = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(mask));
}
// 128-byte swizzled rows along N (the MMA's K runs over rows): lbo = bytes
// between 64-column boxes, sbo = bytes between groups of 8 rows
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = (uint64_t) ((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t) ((lbo >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t) ((sbo >> 4) & 0x3FFFu) << 32;
    d |= (uint64_t) 1u << 46;
    d |= (uint64_t) 2u << 61;
    return d;
}
// 32 columns of a row on their way into f; tmem_ld_wait ends all of a warp's loads
__device__ __forceinline__ void tmem_ld32_begin(uint32_t taddr, float *f) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
          "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]),
          "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]),
          "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16_begin(uint32_t taddr, float *f) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
          "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15])
        : "r"(taddr));
}
// uses of f stay behind the wait above this
__device__ __forceinline__ void tmem_ld32_end(float *f) {
    asm volatile(""
                 : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7]),
                   "+f"(f[8]), "+f"(f[9]), "+f"(f[10]), "+f"(f[11]), "+f"(f[12]), "+f"(f[13]), "+f"(f[14]),
                   "+f"(f[15]));
    asm volatile(""
                 : "+f"(f[16]), "+f"(f[17]), "+f"(f[18]), "+f"(f[19]), "+f"(f[20]), "+f"(f[21]), "+f"(f[22]),
                   "+f"(f[23]), "+f"(f[24]), "+f"(f[25]), "+f"(f[26]), "+f"(f[27]), "+f"(f[28]), "+f"(f[29]),
                   "+f"(f[30]), "+f"(f[31]));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void named_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

// bit c set: column base + c lies in [a, b), c < 32
__device__ __forceinline__ uint32_t bits32(int a, int b, int base) {
    const int lo = min(max(a - base, 0), 32), hi = min(max(b - base, 0), 32);
    const uint32_t below_hi = hi == 32 ? 0xffffffffu : (1u << hi) - 1u;
    const uint32_t below_lo = lo == 32 ? 0xffffffffu : (1u << lo) - 1u;
    return below_hi & ~below_lo;
}

// what a part's sums count for once the maximum is M; a part that saw no key
// has (-inf, 0), one whose scores were NaN a NaN sum
__device__ __forceinline__ float part_factor(float2 ml, float M) {
    return ml.x == -INFINITY ? ml.y : ex2(ml.x - M);
}

// n values of a row that is not aligned, or ends, for a vector store
__device__ __noinline__ void copy_halves(__half *y, const __half *x, int n) {
    for (int i = 0; i < n; i++) y[i] = x[i];
}

template <int DB, bool SPLIT>
__global__ void __launch_bounds__(352, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const __grid_constant__ at_params p) {
    using cfg = at_cfg<DB, SPLIT>;
    constexpr int ST = cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    // SPLIT, once the products are in: (m, sum) of every part's rows, and its O; the rows' places in `out`
    float2 *s_ml = (float2 *) smem;
    int64_t *s_out = (int64_t *) (smem + 2048);
    float *parts = (float *) (smem + cfg::NQ * cfg::Q_BYTES);
    uint64_t *bars = (uint64_t *) (smem + cfg::DATA);
    uint32_t *tmem_slot = (uint32_t *) (bars + cfg::NBARS);
    const uint32_t sq = smem_u32(smem), skv = sq + cfg::NQ * cfg::Q_BYTES;
    auto bar = [&](int i) { return smem_u32(bars + i); };
    auto stage = [&](int s) { return skv + s * cfg::STAGE_BYTES; };
    auto full = [&](int s) { return bar(s); };
    auto empty = [&](int s) { return bar(ST + s); };
    // warpgroup t has two buffers of scores, used in turn: S of buffer x is in
    // TMEM; its P is in TMEM in its place (S read, O rescaled)
    auto s_full = [&](int t, int x) { return bar(2 * ST + 2 * t + x); };
    auto p_full = [&](int t, int x) { return bar(2 * ST + 4 + 2 * t + x); };
    auto o_done = [&](int t, int x) { return bar(2 * ST + 8 + 2 * t + x); };  // O += P V is done
    // the values of keys that no row sees are cleared: at most two tiles a CTA,
    // the window's last and the sinks' last, each with a barrier of its own
    auto v_fixed = [&](int i) { return bar(2 * ST + 12 + i); };
    const uint32_t q_full = bar(2 * ST + 14), fin = bar(2 * ST + 15);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const attn_desc &d = p.d;
    if (threadIdx.x == 32) {
        prefetch_map(&tmQ);
        prefetch_map(&tmK);
        prefetch_map(&tmV);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), SPLIT ? 1 : 2);  // the MMA warps that read the stage
        }
        for (int t = 0; t < 2; t++) {
            for (int x = 0; x < 2; x++) {
                mbar_init(s_full(t, x), 1);
                mbar_init(p_full(t, x), 4);
                mbar_init(o_done(t, x), 1);
            }
        }
        mbar_init(q_full, 1);
        mbar_init(v_fixed(0), 1);
        mbar_init(v_fixed(1), 1);
        mbar_init(fin, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // The set-up runs while the kernel before this one ends. TMEM is had before
    // this one's dependents may start: one that took it first on an SM would wait
    // for this kernel, and this kernel for it.
    pdl_wait();
    pdl_trigger();
    // block -> (cluster rank,) batch and key head, query tile (the last ones,
    // which see most keys, first)
    int idx = blockIdx.x;
    const int rank = SPLIT ? idx % p.splits : 0;
    if (SPLIT) idx /= p.splits;
    const int bh = idx % (d.B * d.Hkv), qt = p.qtiles - 1 - idx / (d.B * d.Hkv);
    const int b = bh / d.Hkv, hk = bh % d.Hkv;
    const int n = d.q_len ? min(max(d.q_len[b], 0), d.Tq) : d.Tq;
    const int L = d.kv_len ? min(max(d.kv_len[b], 0), d.Tk) : d.Tk;
    const int tok0 = qt * p.tb * cfg::NQ;                        // the CTA's first token
    const int toks = min(n - tok0, p.tb * cfg::NQ);              // and how many exist
    auto release = [&] {
        if (warp == 9)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    };
    if (toks <= 0) {  // (the whole cluster alike)
        release();
        return;
    }
    const int64_t pos0 = (int64_t) L - n + tok0;
    const key_range kr = keys_of(d, L, pos0, pos0 + toks - 1);
    // tiles of the window, then of the sinks; SPLIT: this CTA's share of them
    constexpr int KT = cfg::KT;
    const int nwin = (kr.hi - kr.lo + KT - 1) / KT, nall = nwin + (kr.first + KT - 1) / KT;
    const int i0 = SPLIT ? (int) ((int64_t) nall * rank / p.splits) : 0;
    const int nt = (SPLIT ? (int) ((int64_t) nall * (rank + 1) / p.splits) : nall) - i0;
    // (of tile j: its first key, how many of its keys some row sees, and these rounded up for the MMAs)
    const int jwin = nwin - i0;  // the share's first tile of sinks
    auto tile_key = [&](int j) { return j < jwin ? kr.lo + (i0 + j) * KT : (j - jwin) * KT; };
    auto tile_keys = [&](int j) { return min(KT, (j < jwin ? kr.hi : kr.first) - tile_key(j)); };
    auto tile_w = [&](int j) { return (tile_keys(j) + 15) & ~15; };
    // warpgroup t goes through tiles [from, to) and those of the sinks. Prompts:
    // what its rows see of the window (all of it from the start where that
    // begins within the sinks); SPLIT: every other tile
    const int toks0 = min(toks, p.tb), toks1 = toks - toks0;
    int to0 = nt, from1 = 0, to1 = nt;
    if (!SPLIT) {
        const key_range kr0 = keys_of(d, L, pos0, pos0 + toks0 - 1);
        to0 = (kr0.hi - kr.lo + KT - 1) / KT;
        if (toks1 > 0) {
            const key_range kr1 = keys_of(d, L, pos0 + toks0, pos0 + toks - 1);
            from1 = kr.lo < d.sinks ? 0 : (kr1.lo - kr.lo) / KT;
            to1 = (kr1.hi - kr.lo + KT - 1) / KT;
        }
    }
    auto active = [&](int t, int j) {
        if (SPLIT) return (j & 1) == t;
        return t == 0 ? j < to0 || j >= jwin : toks1 > 0 && (j >= from1 && j < to1 || j >= jwin);
    };

    auto t_s = [&](int t, int x) { return tmem + t * 128 + x * KT; };
    auto t_o = [&](int t) { return tmem + 256 + t * DB * 64; };
    bool ok = true;
    // a stage for each step of the MMA warp: first the K of the first AHEAD
    // tiles (two a warpgroup), two a stage, then V(j) with K(j + AHEAD)
    constexpr int AHEAD = SPLIT ? 4 : 2;

    if (warp == 8) {
        int cnt = 0, slot = 0, ph = 0;  // stages so far, the next one's slot and its phase
        auto load = [&](const CUtensorMap *tm0, int j0, const CUtensorMap *tm1, int j1) {  // j1 < nt, or one tile
            if (cnt >= ST && !warp_wait(empty(slot), ph ^ 1)) return false;
            if (elect_one()) {
                mbar_expect_tx(full(slot), j1 < nt ? cfg::STAGE_BYTES : cfg::TILE_BYTES);
#pragma unroll
                for (int x = 0; x < DB; x++)
                    tma_load_4d(stage(slot) + x * (KT * 128), tm0, full(slot), x * 64, tile_key(j0), hk, b);
                if (j1 < nt)
#pragma unroll
                    for (int x = 0; x < DB; x++)
                        tma_load_4d(stage(slot) + cfg::TILE_BYTES + x * (KT * 128), tm1, full(slot), x * 64, tile_key(j1), hk,
                                    b);
            }
            __syncwarp();
            return true;
        };
        auto next = [&] {
            cnt++;
            if (++slot == ST) {
                slot = 0;
                ph ^= 1;
            }
        };
        if (lane == 0 && nt > 0) {
            const uint32_t box = p.tb * p.g * 128;
            mbar_expect_tx(q_full, box * DB * (SPLIT ? p.reps : 2));
            for (int x = 0; x < DB; x++)
                for (int r = 0; r < (SPLIT ? p.reps : 2); r++)
                    tma_load_5d(sq + (SPLIT ? r * (128 / p.reps) * 128 : r * cfg::Q_BYTES) + x * 16384, &tmQ, q_full,
                                x * 64, 0, tok0 + (SPLIT ? 0 : r * p.tb), hk, b);
        }
        __syncwarp();
        for (int e = 0; ok && e < AHEAD / 2; e++) {
            if (e < nt) ok = load(&tmK, e, &tmK, e + AHEAD / 2);
            next();
        }
        for (int j = 0; ok && j < nt; j++) {
            ok = load(&tmV, j, &tmK, j + AHEAD);
            const int keys = tile_keys(j), w = tile_w(j);
            if (ok && keys < w) {
                // values of keys that no row sees: cleared (their weights are zero)
                ok = warp_wait(full(slot), ph);
                if (!ok) break;
                for (int i = lane; i < (w - keys) * 8 * DB; i += 32) {
                    const int x = i / ((w - keys) * 8), o = i % ((w - keys) * 8);
                    *reinterpret_cast<uint4 *>(smem + (stage(slot) - sq) + x * (KT * 128) + keys * 128 + o * 16) =
                        make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(v_fixed(j < jwin ? 0 : 1));
            }
            next();
        }
        // the copies in flight land before the CTA goes on (the first stages are
        // empty where there are fewer tiles than warpgroups)
        for (int i = max(0, cnt - ST); i < cnt; i++)
            if ((i >= AHEAD / 2 || i < nt) && !warp_wait(full(i % ST), (i / ST) & 1)) ok = false;
        if (nt > 0 && !warp_wait(q_full, 0)) ok = false;
        if (!ok && lane == 0) atomicExch(p.err, 1);
    } else if (warp >= 9) {
        // the MMAs of warpgroup t: the whole warp goes through the loop, so that
        // what it computes stays in uniform registers, and one lane issues.
        // (Two warps: what one does between its MMAs, the other's hide.)
        const int t = warp - 9;
        if (nt > 0) {
            // D f32 (bit 4), f16 operands; M >> 4 at bit 24, N >> 3 at bit 17; B along N (bit 16) for V
            const uint32_t id_base = (1u << 4) | (8u << 24);
            const int ksteps = (d.D + 15) / 16;
            const uint32_t id_pv = id_base | (1u << 16) | ((uint32_t) (ksteps * 2) << 17);
            int slot = 0, ph = 0, issued = 0, done = 0;
            auto skip = [&](int n) {  // n < ST stages on
                slot += n;
                if (slot >= ST) {
                    slot -= ST;
                    ph ^= 1;
                }
            };
            const uint64_t aq = smem_desc(sq + (SPLIT ? 0 : t * cfg::Q_BYTES), 1024, 2);
            // (by the elected lane) S of buffer x = Q K^T of a tile of w keys
            auto qk = [&](int x, int w, uint32_t k_tile) {
                const uint64_t bb = smem_desc(k_tile, 1024, 2);
                const uint32_t id = id_base | ((uint32_t) (w >> 3) << 17);
#pragma unroll
                for (int k = 0; k < DB * 4; k++)
                    if (k < ksteps)
                        umma_f16(t_s(t, x), aq + (k >> 2) * 1024 + (k & 3) * 2, bb + (k >> 2) * (KT * 8) + (k & 3) * 2, id,
                                 k > 0);
                umma_commit(s_full(t, x));
            };
            ok = warp_wait(q_full, 0);
            // the first two tiles' scores: SPLIT tiles t and t + 2 in stage t, else 0 and 1 in the only one
            const int first = SPLIT ? t : 0;
            if (SPLIT) skip(t);
            if (ok && first < nt) {
                ok = warp_wait(full(slot), ph);
                if (ok) {
                    tc_fence_after();
                    for (int e = 0; e < 2; e++) {
                        const int j = first + e * (AHEAD / 2);
                        if (j < nt && active(t, j)) {
                            if (elect_one()) qk(issued & 1, tile_w(j), stage(slot) + e * cfg::TILE_BYTES);
                            __syncwarp();
                            issued++;
                        }
                    }
                    if (elect_one()) umma_commit(empty(slot));
                    __syncwarp();
                }
            }
            skip(SPLIT ? 2 : 1);
            for (int j = first; ok && j < nt; j += SPLIT ? 2 : 1) {
                // everything a step needs, then its MMAs without a pause: O += P V
                // of tile j and the scores of tile j + AHEAD
                const int keys = tile_keys(j), w = (keys + 15) & ~15, ja = j + AHEAD, wa = ja < nt ? tile_w(ja) : 0;
                const bool pv = active(t, j), sc = wa > 0 && active(t, ja);
                const int x = done & 1;
                ok = pv ? warp_wait2(full(slot), ph, p_full(t, x), done >> 1 & 1) : warp_wait(full(slot), ph);
                if (ok && keys < w) ok = warp_wait(v_fixed(j < jwin ? 0 : 1), 0);
                if (!ok) break;
                tc_fence_after();
                const uint64_t v = smem_desc_mn(stage(slot), KT * 128, 1024);
                if (elect_one()) {
                    if (pv) {
#pragma unroll
                        for (int k = 0; k < KT / 16; k++)
                            if (k < w / 16)
                                umma_f16_ts(t_o(t), t_s(t, x) + k * 8, v + k * 128, id_pv, done > 0 || k > 0);
                        umma_commit(o_done(t, x));
                    }
                    if (sc) qk(issued & 1, wa, stage(slot) + cfg::TILE_BYTES);
                    umma_commit(empty(slot));
                }
                __syncwarp();
                done += pv;
                issued += sc;
                skip(SPLIT ? 2 : 1);
            }
            // the MMAs in flight end before TMEM is freed
            if (elect_one()) umma_commit(fin);
            __syncwarp();
            if (!warp_wait(fin, 0)) ok = false;
            if (!ok && lane == 0) atomicExch(p.err, 1);
        }
    } else {
        const int t = warp >> 2, q4 = warp & 3;
        const int per = SPLIT ? 128 / p.reps : 128;       // lanes of a copy of the rows
        const int rep = SPLIT ? q4 * 32 / per : 0;
        const int r = q4 * 32 + lane - rep * per;         // row of the tile
        const int tok = tok0 + (SPLIT ? 0 : t * p.tb) + r / p.g, h = hk * p.g + r % p.g;
        const bool row = r < p.tb * p.g && tok < n;
        const bool rows = __any_sync(0xffffffffu, row);
        const key_range kk = keys_of(d, L, (int64_t) L - n + tok, (int64_t) L - n + tok);
        const uint32_t lanes = (uint32_t) (q4 * 32) << 16;
        // the share of each tile's columns that this copy takes, in pieces of 16
        const int c0 = SPLIT ? rep * (4 / p.reps) : 0, c1 = SPLIT ? c0 + 4 / p.reps : 4;
        auto mine = [&](int c) { return !SPLIT || (c >= c0 && c < c1); };
        float m = -INFINITY, l = 0.0f;
        int done = 0;
        for (int j = 0; j < nt; j++) {
            if (!active(t, j)) continue;
            const int buf = done & 1;
            ok = warp_wait(s_full(t, buf), done >> 1 & 1);
            if (!ok) break;
            tc_fence_after();
            if (rows) {
                const uint32_t ts = t_s(t, buf) + lanes;
                const int kb = tile_key(j);
                const bool win = j < jwin;
                // of the window's tiles the row sees [lo, hi) and what lies below
                // sinks, of the sinks' tiles [0, first) below hi
                const int a0 = win ? kk.lo : 0, a1 = win ? kk.hi : min(kr.first, kk.hi);
                const int a2 = win ? min(d.sinks, kk.hi) : 0;
                const bool all = __all_sync(0xffffffffu, a0 <= kb && kb + KT <= a1);
                float s[KT];
                if constexpr (SPLIT) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        if (mine(c)) {
                            tmem_ld16_begin(ts + c * 16, s + c * 16);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; e++) s[c * 16 + e] = -INFINITY;
                        }
                    }
                } else {
                    tmem_ld32_begin(ts, s);
                    tmem_ld32_begin(ts + 32, s + 32);
                }
                tmem_ld_wait();
                tmem_ld32_end(s);
                tmem_ld32_end(s + 32);
                if (!all) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint32_t see = bits32(a0, a1, kb + c * 32) | bits32(0, a2, kb + c * 32);
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (!(see >> e & 1)) s[c * 32 + e] = -INFINITY;
                    }
                }
                float mx[4] = {m, m, m, m};
#pragma unroll
                for (int e = 0; e < KT; e += 2) mx[e >> 1 & 3] = max3(mx[e >> 1 & 3], s[e], s[e + 1]);
                const float mn = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
                // (m - m_old) scale log2(e) above 8, or a first finite maximum
                const bool up = mn > m && !((mn - m) * p.c <= 8.0f);
                if (__any_sync(0xffffffffu, up)) {
                    const float f = up ? ex2((m - mn) * p.c) : 1.0f;
                    if (up) m = mn;
                    l *= f;
                    if (done > 0) {  // O so far, once the last product is in
                        ok = warp_wait(o_done(t, buf ^ 1), (done - 1) >> 1 & 1);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int x = 0; x < DB * 64; x += 16) {
                            uint32_t o[16];
                            tmem_ld16(t_o(t) + lanes + x, o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(t_o(t) + lanes + x, o);
                        }
                        tmem_wait_st();
                    }
                }
                const float mc = m == -INFINITY ? 0.0f : fmaf(m, p.c, -P_EXP);
                const uint64_t c2 = pack2(p.c, p.c), mc2 = pack2(-mc, -mc);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 16) {
                        if (mine(c + e / 16)) {
#pragma unroll
                            for (int i = e; i < e + 16; i += 2) {
                                const float2 x = unpack2(fma2(pack2(s[c * 16 + i], s[c * 16 + i + 1]), c2, mc2));
                                const float x0 = ex2(x.x), x1 = ex2(x.y);
                                sum[i >> 1 & 1] = add2(sum[i >> 1 & 1], pack2(x0, x1));
                                const __half2 hh = __floats2half2_rn(x0, x1);
                                pk[i / 2] = *reinterpret_cast<const uint32_t *>(&hh);
                            }
                        } else {
#pragma unroll
                            for (int i = e; i < e + 16; i += 2) pk[i / 2] = 0;
                        }
                    }
                    tmem_st16(ts + c * 8, pk);
                }
                const float2 s01 = unpack2(add2(sum[0], sum[1]));
                l += s01.x + s01.y;
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(t, buf));
            done++;
        }
        if (ok && done > 0) ok = warp_wait(o_done(t, (done - 1) & 1), (done - 1) >> 1 & 1);
        tc_fence_after();
        if (!ok && lane == 0) atomicExch(p.err, 1);
        if constexpr (!SPLIT) {
            if (nt > 0 && done == 0) ok = warp_wait(q_full, 0);  // (Q lands before its memory is used)
            if (ok && rows) {
                // f16 rows through this warp's part of its Q tile (read for the last
                // time), 16-byte unit u of row i at u ^ (i mod 8) against bank
                // conflicts: a store covers whole rows
                constexpr int UNITS = DB * 8;
                uint8_t *own = smem + t * cfg::Q_BYTES + q4 * 32 * UNITS * 16;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int64_t at = b * d.os[0] + (int64_t) tok * d.os[1] + h * d.os[2];
                // the largest magnitude's bits: above 65504's if it is beyond f16 or NaN
                uint32_t top = 0;
#pragma unroll 1
                for (int x = 0; x < DB * 64; x += 32) {
                    float o[32];
                    if (done > 0) tmem_ld32_begin(t_o(t) + lanes + x, o);
                    tmem_ld_wait();
                    tmem_ld32_end(o);
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        o[e] = done > 0 && x + e < d.D ? o[e] * inv : 0.0f;
                        top = max(top, __float_as_uint(o[e]) & 0x7fffffffu);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        __half2 hh[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) hh[i] = __floats2half2_rn(o[e + 2 * i], o[e + 2 * i + 1]);
                        *reinterpret_cast<uint4 *>(own + lane * UNITS * 16 + (((x + e) / 8) ^ (lane & 7)) * 16) =
                            *reinterpret_cast<const uint4 *>(hh);
                    }
                }
                __syncwarp();
                const int u = lane % UNITS;
#pragma unroll 4
                for (int i0r = 0; i0r < 32; i0r += 32 / UNITS) {
                    const int i = i0r + lane / UNITS;
                    const int64_t off = __shfl_sync(0xffffffffu, at, i);
                    const bool real = __shfl_sync(0xffffffffu, (int) row, i) && u * 8 < d.D;
                    const uint4 *src = reinterpret_cast<const uint4 *>(own + i * UNITS * 16 + (u ^ (i & 7)) * 16);
                    __half *o = (__half *) d.out + off + u * 8;
                    if (real) {
                        if (p.o_vec && u * 8 + 8 <= d.D) *reinterpret_cast<uint4 *>(o) = *src;
                        else copy_halves(o, reinterpret_cast<const __half *>(src), min(8, d.D - u * 8));
                    }
                }
                uint32_t redo = __ballot_sync(0xffffffffu, row && top > 0x477fe000u);
                __syncwarp();
                for (; redo; redo &= redo - 1) {
                    const int src = __ffs(redo) - 1;
                    attn_row<__half, 4>(d, b, __shfl_sync(0xffffffffu, h, src), __shfl_sync(0xffffffffu, tok, src), n, L,
                                        lane);
                }
            }
        } else {
            // join the CTA's parts (part = warpgroup, copy). Each lane scales its
            // part's row by exp(m - M) of the row's maximum M over all parts, and
            // by 1 / sum where no other CTA has parts
            named_sync(1, 256);  // (both warpgroups' products are in: Q and the stages are free)
            const int np = 2 * p.reps, part = t * p.reps + rep;
            if (row) s_ml[part * per + r] = make_float2(m == -INFINITY ? -INFINITY : fmaf(m, p.c, -P_EXP), l);
            named_sync(1, 256);
            if (rows) {
                float M = -INFINITY, sl = 0.0f, f = 0.0f;
                if (row) {
                    for (int k = 0; k < np; k++) M = fmaxf(M, s_ml[k * per + r].x);
                    for (int k = 0; k < np; k++) {
                        const float2 ml = s_ml[k * per + r];
                        sl = fmaf(part_factor(ml, M), ml.y, sl);
                    }
                    f = part_factor(s_ml[part * per + r], M);
                    if (p.splits == 1) f = sl == 0.0f ? 0.0f : f / sl;
                }
#pragma unroll 1
                for (int x = 0; x < DB * 64; x += 32) {
                    float o[32];
                    if (done > 0) {
                        tmem_ld32_begin(t_o(t) + lanes + x, o);
                        tmem_ld_wait();
                        tmem_ld32_end(o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = 0.0f;
                    }
                    if (row) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4 *>(parts + (part * per + r) * cfg::OLD + x + e) =
                                make_float4(o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
                    }
                }
                // (every lane of a row has read s_ml by the next barrier)
                m = M;
                l = sl;
            }
            named_sync(1, 256);
            if (row && part == 0) {
                s_ml[r] = make_float2(m, l);
                s_out[r] = b * d.os[0] + (int64_t) tok * d.os[1] + h * d.os[2];
            }
            named_sync(1, 256);
        }
    }
    if constexpr (SPLIT) {
        // a warp takes a row (two of one box) at a time, four columns a lane
        constexpr int C4 = DB * 16, RPW = 32 / C4;
        const int nrow = min(p.tb, toks) * p.g, np = 2 * p.reps, per = 128 / p.reps, x = lane % C4 * 4;
        auto sum_parts = [&](int rr) {
            float4 o = *reinterpret_cast<const float4 *>(parts + rr * cfg::OLD + x);
            for (int k = 1; k < np; k++) {
                const float4 v = *reinterpret_cast<const float4 *>(parts + (k * per + rr) * cfg::OLD + x);
                o.x += v.x;
                o.y += v.y;
                o.z += v.z;
                o.w += v.w;
            }
            return o;
        };
        // stores a row's four columns; whether one of them is beyond f16 or NaN
        auto put = [&](int rr, float4 o) {
            if (x >= d.D) return false;
            __half *out = (__half *) d.out + s_out[rr] + x;
            const __half2 hh[2] = {__floats2half2_rn(o.x, o.y), __floats2half2_rn(o.z, o.w)};
            if (p.o_vec && x + 4 <= d.D) *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(hh);
            else copy_halves(out, reinterpret_cast<const __half *>(hh), min(4, d.D - x));
            // (columns from D on are zeros, or what is left in TMEM: looked at up to D only)
            const uint32_t a = __float_as_uint(o.x) & 0x7fffffffu, e = __float_as_uint(o.y) & 0x7fffffffu;
            const uint32_t c = __float_as_uint(o.z) & 0x7fffffffu, f = __float_as_uint(o.w) & 0x7fffffffu;
            return max(max(a, x + 1 < d.D ? e : 0u), max(x + 2 < d.D ? c : 0u, x + 3 < d.D ? f : 0u)) > 0x477fe000u;
        };
        uint32_t bad = 0;  // bit i: of this lane's i-th row
        if (p.splits == 1) {
            if (warp < 8) {
                int i = 0;
#pragma unroll 4
                for (int rr = warp * RPW + lane / C4; rr < nrow; rr += 8 * RPW, i++) bad |= (uint32_t) put(rr, sum_parts(rr)) << i;
            }
        } else {
            if (warp < 8)
                for (int rr = warp * RPW + lane / C4; rr < nrow; rr += 8 * RPW)
                    *reinterpret_cast<float4 *>(parts + rr * cfg::OLD + x) = sum_parts(rr);
            cluster_sync_all();
            if (warp < 8) {
                const uint32_t a_ml = smem_u32(s_ml), a_o = smem_u32(parts) + x * 4;
                int i = 0;
#pragma unroll 1
                for (int rr = (rank * 8 + warp) * RPW + lane / C4; rr < nrow; rr += p.splits * 8 * RPW, i++) {
                    float M = -INFINITY, sl = 0.0f;
                    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float2 ml[8];
                    float4 v[8];
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < p.splits) {
                            ml[k] = ld_cluster2(cluster_addr(a_ml + rr * 8, k));
                            v[k] = ld_cluster4(cluster_addr(a_o + rr * cfg::OLD * 4, k));
                            M = fmaxf(M, ml[k].x);
                        }
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < p.splits) {
                            const float f = part_factor(ml[k], M);
                            sl = fmaf(f, ml[k].y, sl);
                            o.x = fmaf(f, v[k].x, o.x);
                            o.y = fmaf(f, v[k].y, o.y);
                            o.z = fmaf(f, v[k].z, o.z);
                            o.w = fmaf(f, v[k].w, o.w);
                        }
                    const float inv = sl == 0.0f ? 0.0f : 1.0f / sl;
                    bad |= (uint32_t) put(rr, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv)) << i;
                }
            }
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, bad != 0))
            for (int i = 0; i < 32; i++)
                for (int e = 0; e < RPW; e++) {
                    const uint32_t of = __ballot_sync(0xffffffffu, bad >> i & 1) & (RPW == 1 ? 0xffffffffu : 0xffffu << 16 * e);
                    if (!of) continue;
                    const int rr = ((p.splits == 1 ? 0 : rank * 8) + warp) * RPW + e + i * (p.splits * 8 * RPW);
                    attn_row<__half, 4>(d, b, hk * p.g + rr % p.g, tok0 + rr / p.g, n, L, lane);
                }
        // no CTA leaves while others read its parts
        if (p.splits > 1) cluster_sync_all();
    }
    tc_fence_before();
    __syncthreads();
    release();
}

// a tensor map over f16 memory: dims and strides (elements) innermost first,
// the innermost contiguous
bool encode_f16(CUtensorMap *tm, const void *base, int rank, const int64_t *dims, const int64_t *strides,
                const int *box) {
    auto enc = encode_fn();
    if (!enc) return false;
    cuuint64_t gd[5], gs[4];
    cuuint32_t bx[5], es[5];
    for (int i = 0; i < rank; i++) {
        gd[i] = (cuuint64_t) dims[i];
        bx[i] = (cuuint32_t) box[i];
        es[i] = 1;
        // a dimension of one element has no stride of its own
        if (i) gs[i - 1] = (cuuint64_t) (dims[i] > 1 ? strides[i] * 2 : 16);
    }
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, (void *) base, gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DB, bool SPLIT>
cudaError_t run_tc(const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV, const at_params &p,
                   unsigned ctas, cudaStream_t st) {
    using cfg = at_cfg<DB, SPLIT>;
    static std::mutex mu;
    static uint64_t attr_set = 0;  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> g(mu);
        if (!(attr_set >> (dev & 63) & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(attn_tc_kernel<DB, SPLIT>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, cfg::SMEM);
            if (e != cudaSuccess) return e;
            attr_set |= 1ull << (dev & 63);
        }
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(ctas, 1, 1);
    lc.blockDim = dim3(cfg::THREADS, 1, 1);
    lc.dynamicSmemBytes = cfg::SMEM;
    lc.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned) p.splits;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = p.splits > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&lc, attn_tc_kernel<DB, SPLIT>, tmQ, tmK, tmV, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// whether TMA can address a tensor: 16-byte aligned base and strides, no
// stride of 0 or backwards over more than one element
bool tma_ok(const void *base, const int64_t *s, int64_t n0, int64_t n1, int64_t n2) {
    const int64_t dim[3] = {n0, n1, n2};
    if ((uintptr_t) base & 15) return false;
    for (int i = 0; i < 3; i++)
        if (dim[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= 1ll << 38)) return false;
    return true;
}

}  // namespace

bool attn_tc_supported(const attn_desc &d) {
    return d.f16 && d.D <= 128 && d.Tk > 0 && d.Hq / d.Hkv <= 128 && d.scale > 0.0f &&
           tma_ok(d.q, d.qs, d.B, d.Tq, d.Hq) && tma_ok(d.k, d.ks, d.B, d.Tk, d.Hkv) &&
           tma_ok(d.v, d.vs, d.B, d.Tk, d.Hkv) && d.qs[2] * (d.Hq / d.Hkv) < 1ll << 38;
}

cudaError_t launch_attn_tc(const attn_desc &d, cudaStream_t st) {
    at_params p{};
    p.d = d;
    p.g = d.Hq / d.Hkv;
    p.c = d.scale * 1.4426950408889634f;
    p.o_vec = !((uintptr_t) d.out & 15) && (d.B == 1 || d.os[0] % 8 == 0) && (d.Tq == 1 || d.os[1] % 8 == 0) &&
              (d.Hq == 1 || d.os[2] % 8 == 0);
    p.err = d.err ? d.err : tpk_err_word();
    if (!p.err) return cudaErrorUnknown;
    const int64_t bh = (int64_t) d.B * d.Hkv;
    const int sms = sm_count(), tb = 128 / p.g;
    // two row tiles a CTA where that fills the SMs; otherwise one, its keys
    // shared out over both warpgroups and a cluster
    const bool split = bh * ((d.Tq + 2 * tb - 1) / (2 * tb)) < sms;
    p.tb = split ? std::min(tb, d.Tq) : tb;
    const int rows = p.tb * p.g;
    p.reps = !split || rows > 64 ? 1 : rows > 32 ? 2 : 4;
    const int per_cta = split ? p.tb : 2 * p.tb;
    p.qtiles = (d.Tq + per_cta - 1) / per_cta;
    p.splits = 1;
    if (split) {
        int64_t keys = d.Tk;
        if (d.left >= 0 && d.right >= 0) keys = std::min<int64_t>(keys, (int64_t) p.tb + d.left + d.right + d.sinks);
        const int64_t tiles = (keys + 63) / 64, ctas = bh * p.qtiles;
        p.splits = cluster_size(ctas, (tiles + 3) / 4);
    }
    const int64_t ctas = bh * p.qtiles * p.splits;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    CUtensorMap tmQ, tmK, tmV;
    const int64_t qd[5] = {d.D, p.g, d.Tq, d.Hkv, d.B}, qs[5] = {1, d.qs[2], d.qs[1], d.qs[2] * p.g, d.qs[0]};
    const int64_t kd[4] = {d.D, d.Tk, d.Hkv, d.B};
    const int64_t ks[4] = {1, d.ks[1], d.ks[2], d.ks[0]}, vs[4] = {1, d.vs[1], d.vs[2], d.vs[0]};
    const int qb[5] = {64, p.g, p.tb, 1, 1}, kb[4] = {64, 64, 1, 1};
    if (!encode_f16(&tmQ, d.q, 5, qd, qs, qb) || !encode_f16(&tmK, d.k, 4, kd, ks, kb) ||
        !encode_f16(&tmV, d.v, 4, kd, vs, kb))
        return cudaErrorInvalidValue;
    const unsigned n = (unsigned) ctas;
    if (d.D <= 64)
        return split ? run_tc<1, true>(tmQ, tmK, tmV, p, n, st) : run_tc<1, false>(tmQ, tmK, tmV, p, n, st);
    return split ? run_tc<2, true>(tmQ, tmK, tmV, p, n, st) : run_tc<2, false>(tmQ, tmK, tmV, p, n, st);
}

}  // namespace tpmd
