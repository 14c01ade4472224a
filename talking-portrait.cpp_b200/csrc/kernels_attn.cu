// Sliding-window attention with first tokens that stay visible
// (tpk_attn_window, include/tpmd.h): the entry point, and the form on the CUDA
// cores in f32, for f32 inputs (the parity type) and for whatever the
// tensor-core form does not take (head widths above 128, rows that TMA cannot
// address).
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max),
//   over keys j < min(L, p + right + 1) with j >= p - left or j < sinks,
//   p = L - n + i
//
// Rows are tokens times the query heads of a group, so that these share a key
// head's tiles; the keys that any row of a CTA sees are one list, the sinks
// and the window behind them, in tiles with a running maximum and sum. K and
// V tiles come by cp.async. Two kernels:
//
//  * attn_tile_kernel, many rows: 64 a CTA, tiles of 32 keys, one ahead.
//    Thread (rg, kx) = (tid / 8, tid % 8) has rows rg + 16 j: their scores
//    with keys kx + 8 i, then columns 4 kx + 32 i of their outputs (register
//    tiles of 4 x 4 RPT). Bound by shared-memory reads and FMAs alike, half
//    of either's rate with the eight warps that fit an SM: 30 TFLOP/s (4096
//    tokens, 16 heads of 128 on 4, 1024 keys each, 1.02 ms).
//  * attn_rows_kernel, few rows: up to 16 a CTA. Every warp has all rows and
//    its own share of the keys, its own tiles (8 keys, K and V two ahead) and
//    nothing to wait for but its copies; lane (rg, kx) as above with rows
//    rg + 4 j. The warps' parts join in shared memory, and where CTAs do not
//    fill the SMs a cluster of up to eight shares the keys and joins over
//    distributed shared memory; always in the same order. Bound by the
//    latency of shared-memory reads: 268 MB of cache in 73 us, 3.7 TB/s (16
//    sequences of one token, 16 heads of 128 on 4, 4100 keys); the sampler's
//    60 frames of 3 x 8 heads over 5 + 10 keys in 9.4 us, 2.5 of them a
//    launch.
//
// Values of keys that no row sees load as zeros; a row that comes out not
// finite is computed again from its visible keys alone (a weight of zero
// times a value that is not finite is NaN).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "../../include/tpmd.h"
#include "attn_row.cuh"
#include "tc_ptx.cuh"
#include "tpmd_internal.h"

namespace tpmd {
namespace {

struct tile_params {
    attn_desc d;
    int g, qtiles, splits;
    float c;  // scale log2(e)
    bool q_vec, kv_vec;  // four elements of q, of k and v, load at once
};

__device__ __forceinline__ float4 load4(const float *x, int n, bool vec) {
    if (vec && n >= 4) return *reinterpret_cast<const float4 *>(x);
    return make_float4(n > 0 ? x[0] : 0.0f, n > 1 ? x[1] : 0.0f, n > 2 ? x[2] : 0.0f, n > 3 ? x[3] : 0.0f);
}
__device__ __forceinline__ float4 load4(const __half *x, int n, bool vec) {
    if (vec && n >= 4) {
        const uint2 t = *reinterpret_cast<const uint2 *>(x);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&t.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&t.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(n > 0 ? __half2float(x[0]) : 0.0f, n > 1 ? __half2float(x[1]) : 0.0f,
                       n > 2 ? __half2float(x[2]) : 0.0f, n > 3 ? __half2float(x[3]) : 0.0f);
}
__device__ __forceinline__ float dot4(float4 a, float4 b, float s) {
    return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s))));
}

// the sum of n parts of a row, each relative to its own maximum, relative to
// the largest; a lane has columns lane + 32 x
template <int DC, typename ML, typename V>
__device__ __forceinline__ float2 join_parts(int n, ML ml, V part, float (&v)[DC]) {
    float M = -INFINITY, sl = 0.0f;
    for (int k = 0; k < n; k++) M = fmaxf(M, ml(k).x);
#pragma unroll
    for (int x = 0; x < DC; x++) v[x] = 0.0f;
    for (int k = 0; k < n; k++) {
        const float2 t = ml(k);
        const float f = t.x == -INFINITY ? t.y : exp2f(t.x - M);  // (a part that saw no key: 0; NaN stays)
        sl = fmaf(f, t.y, sl);
#pragma unroll
        for (int x = 0; x < DC; x++) v[x] = fmaf(f, part(k, x), v[x]);
    }
    return make_float2(M, sl);
}
// row (token, head of the group) `row` of the outputs from its sums
template <typename T, int DC>
__device__ __forceinline__ void store_row(const tile_params &p, int b, int hk, int64_t row, int n, int L, float sl,
                                          const float (&v)[DC], int lane) {
    const attn_desc &d = p.d;
    const int tok = (int) (row / p.g), h = hk * p.g + (int) (row % p.g);
    T *out = (T *) d.out + b * d.os[0] + tok * d.os[1] + h * d.os[2];
    bool bad = false;
#pragma unroll
    for (int x = 0; x < DC; x++) {
        const int e = lane + 32 * x;
        if (e < d.D) {
            const float y = sl == 0.0f ? 0.0f : v[x] / sl;
            out[e] = from_f<T>(y);
            bad = bad || !(fabsf(y) <= 3.4028235e38f);
        }
    }
    if (__any_sync(0xffffffffu, bad)) attn_row<T, DC>(d, b, h, tok, n, L, lane);
}

// KT rows from number `at` of the list of visible keys (`keys` long: the first
// kr.first, then kr.lo and on) of K or V into shared memory, LD floats apart,
// by THREADS threads; zeros behind the list's end and columns D
template <typename T, int DC, int KT, int LD, int THREADS>
__device__ __forceinline__ void load_keys(const T *src, int64_t stride, int at, const key_range &kr, int keys, int D,
                                          bool vec, float *to, int tid) {
    constexpr int COLS = THREADS < DC * 8 ? THREADS : DC * 8, ROWS = THREADS / COLS;  // of one step, columns of four
    auto key_at = [&](int i) { return i < kr.first ? i : i - kr.first + kr.lo; };
    const int c = tid % COLS * 4, r0 = tid / COLS;
    if (sizeof(T) == 4 && vec && D % 4 == 0 && at + KT <= keys && (at >= kr.first || at + KT <= kr.first)) {
        const T *s = src + (int64_t) (key_at(at) + r0) * stride;
        uint32_t dst = smem_u32(to + r0 * LD + c);
#pragma unroll
        for (int r = 0; r < KT; r += ROWS) {
#pragma unroll
            for (int x = 0; x < DC * 32; x += COLS * 4)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + x * 4),
                             "l"(s + min(c + x, D - 4)), "r"(c + x < D ? 16 : 0)  // 0: zeros, nothing is read
                             : "memory");
            s += ROWS * stride;
            dst += ROWS * LD * 4;
        }
    } else {
        for (int r = r0; r < KT; r += ROWS)
            for (int x = c; x < DC * 32; x += COLS * 4) {
                const int left = at + r < keys ? D - x : 0;
                const T *s = src + (int64_t) key_at(at + r) * stride + x;
                if (sizeof(T) == 4 && vec && (left >= 4 || left <= 0))
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + r * LD + x)),
                                 "l"(left > 0 ? s : src), "r"(left > 0 ? 16 : 0)
                                 : "memory");
                else
                    *reinterpret_cast<float4 *>(to + r * LD + x) = load4(s, left, vec);
            }
    }
}

template <int DC, int RPT>
struct tile_cfg {
    static constexpr int BM = 16 * RPT, KT = 32, DP = 32 * DC, LD = DP + 4, PLD = KT + 4;
    static constexpr int KV = KT * LD;  // floats a K or V tile
    static constexpr int SMEM = (BM * LD + 4 * KV + BM * PLD + BM) * 4;
    static_assert(BM * LD <= 4 * KV, "the sums fit the tiles");
    static_assert(SMEM <= 232448, "shared memory");
};

template <typename T, int DC, int RPT>
__global__ void __launch_bounds__(128)
attn_tile_kernel(const __grid_constant__ tile_params p) {
    using cfg = tile_cfg<DC, RPT>;
    constexpr int KT = cfg::KT, LD = cfg::LD;
    extern __shared__ float4 smem4[];
    float *sq = (float *) smem4, *skv = sq + cfg::BM * LD, *sp = skv + 4 * cfg::KV;
    float *s_l = sp + cfg::BM * cfg::PLD;
    const attn_desc &d = p.d;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, kx = tid % 8, rg = tid / 8;
    const int idx = blockIdx.x;
    const int bh = idx % (d.B * d.Hkv), qt = p.qtiles - 1 - idx / (d.B * d.Hkv);  // (the last rows see most keys)
    const int b = bh / d.Hkv, hk = bh % d.Hkv;
    const int n = d.q_len ? min(max(__ldg(d.q_len + b), 0), d.Tq) : d.Tq;
    const int L = d.kv_len ? min(max(__ldg(d.kv_len + b), 0), d.Tk) : d.Tk;
    const int64_t r0 = (int64_t) qt * cfg::BM;  // rows: token g + head of the group
    const int rows = (int) min((int64_t) cfg::BM, (int64_t) n * p.g - r0);
    if (rows <= 0) return;
    const int64_t base = (int64_t) L - n;
    const key_range kr = keys_of(d, L, base + r0 / p.g, base + (r0 + rows - 1) / p.g);
    // the keys that some row sees, in one list: the sinks, then the window
    const int keys = kr.first + kr.hi - kr.lo, nall = (keys + KT - 1) / KT;
    auto key_at = [&](int i) { return i < kr.first ? i : i - kr.first + kr.lo; };
    const T *kbase = (const T *) d.k + b * d.ks[0] + hk * d.ks[2], *vbase = (const T *) d.v + b * d.vs[0] + hk * d.vs[2];

    for (int i = tid; i < cfg::BM * DC * 8; i += 128) {
        const int r = i / (DC * 8), x = i % (DC * 8) * 4;
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < rows) {
            const int tok = (int) ((r0 + r) / p.g), h = hk * p.g + (int) ((r0 + r) % p.g);
            f = load4((const T *) d.q + b * d.qs[0] + tok * d.qs[1] + h * d.qs[2] + x, d.D - x, p.q_vec);
        }
        *reinterpret_cast<float4 *>(sq + r * LD + x) = make_float4(f.x * p.c, f.y * p.c, f.z * p.c, f.w * p.c);
    }
    auto load = [&](int i) {  // tile i of the list into buffer i & 1
        float *k = skv + (i & 1) * 2 * cfg::KV;
        load_keys<T, DC, KT, LD, 128>(kbase, d.ks[1], i * KT, kr, keys, d.D, p.kv_vec, k, tid);
        load_keys<T, DC, KT, LD, 128>(vbase, d.vs[1], i * KT, kr, keys, d.D, p.kv_vec, k + cfg::KV, tid);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    key_range kk[RPT];
    float m[RPT], l[RPT];
    float4 o[RPT][DC];
#pragma unroll
    for (int j = 0; j < RPT; j++) {
        const int64_t pos = base + (r0 + min(rg + 16 * j, rows - 1)) / p.g;
        kk[j] = keys_of(d, L, pos, pos);
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < DC; i++) o[j][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (nall) load(0);
    for (int i = 0; i < nall; i++) {
        if (i + 1 < nall) {
            load(i + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        const float *k = skv + (i & 1) * 2 * cfg::KV, *v = k + cfg::KV;
        const int here = min(KT, keys - i * KT);  // keys of the tile
        float s[RPT][4];
#pragma unroll
        for (int j = 0; j < RPT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[j][e] = 0.0f;
#pragma unroll 4
        for (int x = 0; x < cfg::DP; x += 4) {
            float4 kv[4];
#pragma unroll
            for (int e = 0; e < 4; e++) kv[e] = *reinterpret_cast<const float4 *>(k + (kx + 8 * e) * LD + x);
#pragma unroll
            for (int j = 0; j < RPT; j++) {
                const float4 q = *reinterpret_cast<const float4 *>(sq + (rg + 16 * j) * LD + x);
#pragma unroll
                for (int e = 0; e < 4; e++) s[j][e] = dot4(q, kv[e], s[j][e]);
            }
        }
#pragma unroll
        for (int j = 0; j < RPT; j++) {
            float mn = m[j];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = kx + 8 * e, key = key_at(i * KT + at);
                if (!(at < here && key < kk[j].hi && (key >= kk[j].lo || key < d.sinks))) s[j][e] = -INFINITY;
                mn = fmaxf(mn, s[j][e]);
            }
#pragma unroll
            for (int w = 4; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
            const float zero = mn == -INFINITY ? 0.0f : mn, f = exp2f(m[j] - zero);
            m[j] = mn;
            l[j] *= f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float w = exp2f(s[j][e] - zero);
                l[j] += w;
                sp[(rg + 16 * j) * cfg::PLD + kx + 8 * e] = w;
            }
#pragma unroll
            for (int e = 0; e < DC; e++) {
                o[j][e].x *= f;
                o[j][e].y *= f;
                o[j][e].z *= f;
                o[j][e].w *= f;
            }
        }
        __syncwarp();  // (a row's weights are written and read by one warp)
#pragma unroll 2
        for (int key = 0; key < here; key += 4) {  // (weights behind the list's end are zeros, and so are the values)
            float4 w[RPT];
#pragma unroll
            for (int j = 0; j < RPT; j++)
                w[j] = *reinterpret_cast<const float4 *>(sp + (rg + 16 * j) * cfg::PLD + key);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int x = 0; x < DC; x++) {
                    const float4 vv = *reinterpret_cast<const float4 *>(v + (key + e) * LD + 4 * kx + 32 * x);
#pragma unroll
                    for (int j = 0; j < RPT; j++) {
                        const float f = e == 0 ? w[j].x : e == 1 ? w[j].y : e == 2 ? w[j].z : w[j].w;
                        o[j][x].x = fmaf(f, vv.x, o[j][x].x);
                        o[j][x].y = fmaf(f, vv.y, o[j][x].y);
                        o[j][x].z = fmaf(f, vv.z, o[j][x].z);
                        o[j][x].w = fmaf(f, vv.w, o[j][x].w);
                    }
                }
        }
        __syncthreads();  // (the tile's buffer is loaded again)
    }
    // sums to shared memory (in the tiles' place), then a row at a time to a warp
#pragma unroll
    for (int j = 0; j < RPT; j++) {
#pragma unroll
        for (int w = 4; w > 0; w >>= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], w);
        const int r = rg + 16 * j;
        if (kx == 0) s_l[r] = l[j];
#pragma unroll
        for (int x = 0; x < DC; x++) *reinterpret_cast<float4 *>(skv + r * LD + 4 * kx + 32 * x) = o[j][x];
    }
    __syncthreads();
    const int lane = tid & 31, warp = tid >> 5;
    for (int r = warp; r < rows; r += 4) {
        float v[DC];
#pragma unroll
        for (int x = 0; x < DC; x++) v[x] = skv[r * LD + lane + 32 * x];
        store_row<T, DC>(p, b, hk, r0 + r, n, L, s_l[r], v, lane);
    }
}

template <int DC, int R, int W>
struct row_cfg {
    static constexpr int WARPS = W, KT = 8, KPL = KT / 8;
    static constexpr int BM = 4 * R, LD = 32 * DC + 4, PLD = KT + 4;
    static constexpr int KV = KT * LD;                  // floats a K or V tile
    static constexpr int WARP = 4 * KV + BM * PLD;      // floats a warp: two tiles of each, weights
    static constexpr int SMEM = (BM * LD + WARPS * WARP + 2 * WARPS * BM) * 4;
    static_assert(BM <= 4 * KT, "a part fits the tiles");
    static_assert(SMEM <= 232448, "shared memory");
};

// few rows: 4 R of them, all by each of the CTA's warps, which share the
// keys out and run on their own until they join
template <typename T, int DC, int R, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
attn_rows_kernel(const __grid_constant__ tile_params p) {
    using cfg = row_cfg<DC, R, WARPS>;
    constexpr int KT = cfg::KT, LD = cfg::LD, KPL = cfg::KPL, BM = cfg::BM;
    extern __shared__ float4 smem4[];
    const attn_desc &d = p.d;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kx = lane % 8, rg = lane / 8;
    float *sq = (float *) smem4, *parts = sq + BM * LD, *skv = parts + warp * cfg::WARP, *sp = skv + 4 * cfg::KV;
    float2 *s_ml = (float2 *) (parts + WARPS * cfg::WARP);
    int idx = blockIdx.x;
    const int rank = idx % p.splits;
    idx /= p.splits;
    const int bh = idx % (d.B * d.Hkv), qt = p.qtiles - 1 - idx / (d.B * d.Hkv);
    const int b = bh / d.Hkv, hk = bh % d.Hkv;
    const int n = d.q_len ? min(max(__ldg(d.q_len + b), 0), d.Tq) : d.Tq;
    const int L = d.kv_len ? min(max(__ldg(d.kv_len + b), 0), d.Tk) : d.Tk;
    const int64_t r0 = (int64_t) qt * BM;
    const int rows = (int) min((int64_t) BM, (int64_t) n * p.g - r0);
    if (rows <= 0) return;  // (the whole cluster alike)
    const int64_t base = (int64_t) L - n;
    const key_range kr = keys_of(d, L, base + r0 / p.g, base + (r0 + rows - 1) / p.g);
    const int keys = kr.first + kr.hi - kr.lo, nall = (keys + KT - 1) / KT;
    auto key_at = [&](int i) { return i < kr.first ? i : i - kr.first + kr.lo; };
    const int share = rank * WARPS + warp, shares = p.splits * WARPS;
    const int i0 = (int) ((int64_t) nall * share / shares), i1 = (int) ((int64_t) nall * (share + 1) / shares);
    // tile i of the list's keys or values into buffer i & 1; always one group
    auto load = [&](int i, const void *tensor, const int64_t *st, float *to) {
        if (i < i1)
            load_keys<T, DC, KT, LD, 32>((const T *) tensor + b * st[0] + hk * st[2], st[1], i * KT, kr, keys, d.D,
                                         p.kv_vec, to, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto load_k = [&](int i) { load(i, d.k, d.ks, skv + (i & 1) * cfg::KV); };
    auto load_v = [&](int i) { load(i, d.v, d.vs, skv + (2 + (i & 1)) * cfg::KV); };
    load_k(i0);
    load_v(i0);
    load_k(i0 + 1);
    load_v(i0 + 1);
    for (int i = tid; i < BM * DC * 8; i += WARPS * 32) {
        const int r = i / (DC * 8), x = i % (DC * 8) * 4;
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < rows) {
            const int tok = (int) ((r0 + r) / p.g), h = hk * p.g + (int) ((r0 + r) % p.g);
            f = load4((const T *) d.q + b * d.qs[0] + tok * d.qs[1] + h * d.qs[2] + x, d.D - x, p.q_vec);
        }
        *reinterpret_cast<float4 *>(sq + r * LD + x) = make_float4(f.x * p.c, f.y * p.c, f.z * p.c, f.w * p.c);
    }
    key_range kk[R];
    float m[R], l[R];
    uint64_t o[R][DC][2];  // pairs of columns
#pragma unroll
    for (int j = 0; j < R; j++) {
        const int64_t pos = base + (r0 + min(rg + 4 * j, rows - 1)) / p.g;
        kk[j] = keys_of(d, L, pos, pos);
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < DC; i++) o[j][i][0] = o[j][i][1] = 0;
    }
    __syncthreads();
    for (int i = i0; i < i1; i++) {
        const float *k = skv + (i & 1) * cfg::KV, *v = skv + (2 + (i & 1)) * cfg::KV;
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        __syncwarp();
        const int here = min(KT, keys - i * KT);  // keys of the tile
        uint64_t s2[R][KPL][2];  // pairs of partial sums
#pragma unroll
        for (int j = 0; j < R; j++)
#pragma unroll
            for (int e = 0; e < KPL; e++) s2[j][e][0] = s2[j][e][1] = 0;
#pragma unroll 8
        for (int x = 0; x < 32 * DC; x += 4) {
            ulonglong2 kv[KPL];
#pragma unroll
            for (int e = 0; e < KPL; e++) kv[e] = *reinterpret_cast<const ulonglong2 *>(k + (kx + 8 * e) * LD + x);
#pragma unroll
            for (int j = 0; j < R; j++) {
                const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(sq + (rg + 4 * j) * LD + x);
#pragma unroll
                for (int e = 0; e < KPL; e++) {
                    s2[j][e][0] = fma2(q.x, kv[e].x, s2[j][e][0]);
                    s2[j][e][1] = fma2(q.y, kv[e].y, s2[j][e][1]);
                }
            }
        }
        __syncwarp();  // (K's buffer is loaded again)
        load_k(i + 2);
#pragma unroll
        for (int j = 0; j < R; j++) {
            float s[KPL], mn = m[j];
#pragma unroll
            for (int e = 0; e < KPL; e++) {
                const int at = kx + 8 * e, key = key_at(i * KT + at);
                const float2 h = unpack2(add2(s2[j][e][0], s2[j][e][1]));
                s[e] = at < here && key < kk[j].hi && (key >= kk[j].lo || key < d.sinks) ? h.x + h.y : -INFINITY;
                mn = fmaxf(mn, s[e]);
            }
#pragma unroll
            for (int w = 4; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
            const float zero = mn == -INFINITY ? 0.0f : mn, f = exp2f(m[j] - zero);
            m[j] = mn;
            l[j] *= f;
#pragma unroll
            for (int e = 0; e < KPL; e++) {
                const float w = exp2f(s[e] - zero);
                l[j] += w;
                sp[(rg + 4 * j) * cfg::PLD + kx + 8 * e] = w;
            }
            const uint64_t ff = pack2(f, f);
#pragma unroll
            for (int e = 0; e < DC; e++)
#pragma unroll
                for (int y = 0; y < 2; y++) o[j][e][y] = mul2(o[j][e][y], ff);
        }
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        __syncwarp();
        for (int key = 0; key < here; key += 4) {  // (weights behind the list's end are zeros, and so are the values)
            float4 w[R];
#pragma unroll
            for (int j = 0; j < R; j++) w[j] = *reinterpret_cast<const float4 *>(sp + (rg + 4 * j) * cfg::PLD + key);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint64_t ww[R];
#pragma unroll
                for (int j = 0; j < R; j++) {
                    const float f = e == 0 ? w[j].x : e == 1 ? w[j].y : e == 2 ? w[j].z : w[j].w;
                    ww[j] = pack2(f, f);
                }
#pragma unroll
                for (int x = 0; x < DC; x++) {
                    const ulonglong2 vv = *reinterpret_cast<const ulonglong2 *>(v + (key + e) * LD + 4 * kx + 32 * x);
#pragma unroll
                    for (int j = 0; j < R; j++) {
                        o[j][x][0] = fma2(ww[j], vv.x, o[j][x][0]);
                        o[j][x][1] = fma2(ww[j], vv.y, o[j][x][1]);
                    }
                }
            }
        }
        __syncwarp();  // (V's buffer and the weights are written again)
        load_v(i + 2);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // parts to shared memory in the tiles' place; the CTA's join in the
    // first one's, then the cluster's
#pragma unroll
    for (int j = 0; j < R; j++) {
#pragma unroll
        for (int w = 4; w > 0; w >>= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], w);
        const int r = rg + 4 * j;
        if (kx == 0) s_ml[warp * BM + r] = make_float2(m[j], l[j]);
#pragma unroll
        for (int x = 0; x < DC; x++) *reinterpret_cast<ulonglong2 *>(skv + r * LD + 4 * kx + 32 * x) = make_ulonglong2(o[j][x][0], o[j][x][1]);
    }
    __syncthreads();
    for (int r = warp; r < rows; r += WARPS) {
        float v[DC];
        const float2 ml = join_parts<DC>(
            WARPS, [&](int k) { return s_ml[k * BM + r]; },
            [&](int k, int x) { return parts[k * cfg::WARP + r * LD + lane + 32 * x]; }, v);
        if (p.splits == 1) {
            store_row<T, DC>(p, b, hk, r0 + r, n, L, ml.y, v, lane);
        } else {
            __syncwarp();  // (every lane has read them)
            if (lane == 0) s_ml[r] = ml;
#pragma unroll
            for (int x = 0; x < DC; x++) parts[r * LD + lane + 32 * x] = v[x];
        }
    }
    if (p.splits == 1) return;
    cluster_sync_all();
    for (int r = rank * WARPS + warp; r < rows; r += p.splits * WARPS) {
        float v[DC];
        const float2 ml = join_parts<DC>(
            p.splits,
            [&](int k) { return make_float2(ld_part(&s_ml[r].x, k, p.splits), ld_part(&s_ml[r].y, k, p.splits)); },
            [&](int k, int x) { return ld_part(parts + r * LD + lane + 32 * x, k, p.splits); }, v);
        store_row<T, DC>(p, b, hk, r0 + r, n, L, ml.y, v, lane);
    }
    cluster_sync_all();  // no CTA leaves while others read its parts
}

template <auto kernel>
cudaError_t launch(tile_params &p, int rows, int threads, int smem, int64_t most_splits, cudaStream_t st) {
    const attn_desc &d = p.d;
    const int64_t qtiles = ((int64_t) d.Tq * p.g + rows - 1) / rows, bh = (int64_t) d.B * d.Hkv;
    if (qtiles > INT32_MAX || bh * qtiles > INT32_MAX / 8) return cudaErrorInvalidValue;
    p.qtiles = (int) qtiles;
    p.splits = cluster_size(bh * qtiles, most_splits);
    static std::mutex mu;
    static uint64_t attr_set = 0;  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> g(mu);
        if (!(attr_set >> (dev & 63) & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) return e;
            attr_set |= 1ull << (dev & 63);
        }
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned) (bh * qtiles * p.splits), 1, 1);
    lc.blockDim = dim3(threads, 1, 1);
    lc.dynamicSmemBytes = smem;
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
    const cudaError_t e = cudaLaunchKernelEx(&lc, kernel, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int DC, int R, int WARPS>
cudaError_t run_warps(tile_params &p, cudaStream_t st) {
    using cfg = row_cfg<DC, R, WARPS>;
    const attn_desc &d = p.d;
    // the keys that a CTA's rows can see
    int64_t keys = d.Tk;
    if (d.left >= 0 && d.right >= 0)
        keys = std::min<int64_t>(keys, cfg::BM / p.g + 2 + (int64_t) d.left + d.right + d.sinks);
    // parts down to a tile of keys a warp
    const int64_t most = (keys + WARPS * cfg::KT - 1) / (WARPS * cfg::KT);
    return launch<attn_rows_kernel<T, DC, R, WARPS>>(p, cfg::BM, WARPS * 32, cfg::SMEM, most, st);
}

template <typename T, int DC, int R>
cudaError_t run_few(tile_params &p, cudaStream_t st) {
    // eight warps a CTA hide more of each other's latency; with four, three
    // CTAs fit an SM and one's start and end hide behind the others (768
    // rows of 128 over 200 keys each 69 -> 44 us; four rows over 4100 keys,
    // 64 times, 73 us against 110)
    const int64_t ctas = ((int64_t) p.d.Tq * p.g + 4 * R - 1) / (4 * R) * p.d.B * p.d.Hkv;
    if (DC > 4 || ctas >= 2 * sm_count()) return run_warps<T, DC, R, 4>(p, st);
    return run_warps<T, DC, R, (DC > 4 ? 4 : 8)>(p, st);
}

template <typename T, int DC>
cudaError_t run_rows(tile_params &p, cudaStream_t st) {
    // 64 rows a CTA (32 of wide heads) where that fills the SMs and more than
    // half of the tiles (64 sequences of 12 heads of 128, 500 keys: of 32 rows
    // 453 us in tiles, 271 in 16 rows a CTA; of 48 rows 464, 475)
    constexpr int RPT = DC > 4 ? 2 : 4;
    const int64_t rows = (int64_t) p.d.Tq * p.g, tiles = (rows + 16 * RPT - 1) / (16 * RPT) * p.d.B * p.d.Hkv;
    if (rows > 8 * RPT && tiles >= sm_count())
        return launch<attn_tile_kernel<T, DC, RPT>>(p, 16 * RPT, 128, tile_cfg<DC, RPT>::SMEM, 1, st);
    return rows <= 4 ? run_few<T, DC, 1>(p, st) : rows <= 8 ? run_few<T, DC, 2>(p, st) : run_few<T, DC, 4>(p, st);
}

template <typename T>
cudaError_t run_simt(const attn_desc &d, cudaStream_t st) {
    tile_params p{};
    p.d = d;
    p.g = d.Hq / d.Hkv;
    p.c = d.scale * 1.4426950408889634f;
    auto vec = [&](const void *x, const int64_t *s, int64_t n1, int64_t n2) {
        return !((uintptr_t) x & (4 * sizeof(T) - 1)) && (d.B == 1 || s[0] % 4 == 0) && (n1 <= 1 || s[1] % 4 == 0) &&
               (n2 <= 1 || s[2] % 4 == 0);
    };
    p.q_vec = vec(d.q, d.qs, d.Tq, d.Hq);
    p.kv_vec = vec(d.k, d.ks, d.Tk, d.Hkv) && vec(d.v, d.vs, d.Tk, d.Hkv);
    if (d.D <= 64) return run_rows<T, 2>(p, st);
    if (d.D <= 128) return run_rows<T, 4>(p, st);
    return run_rows<T, 8>(p, st);
}

// whether every output element has an address of its own: from the smallest
// stride up, each steps over everything that the ones before it span
bool own_rows(const int64_t *stride, int64_t n0, int64_t n1, int64_t n2, int64_t D) {
    std::pair<int64_t, int64_t> d[3] = {{stride[0], n0}, {stride[1], n1}, {stride[2], n2}};
    for (auto &x : d) x.first = x.first < 0 ? -x.first : x.first;
    std::sort(d, d + 3);
    int64_t span = D;
    for (auto &x : d) {
        if (x.second <= 1) continue;
        if (x.first < span) return false;
        span += x.first * (x.second - 1);
    }
    return true;
}

}  // namespace

cudaError_t launch_attn(const attn_desc &d, cudaStream_t st) {
    if (d.D < 1 || d.D > 256) return cudaErrorInvalidValue;
    if (attn_tc_supported(d)) return launch_attn_tc(d, st);
    return d.f16 ? run_simt<__half>(d, st) : run_simt<float>(d, st);
}

}  // namespace tpmd

extern "C" int tpk_attn_window(const void *q, const void *k, const void *v, void *out, const int64_t strides[12],
                               int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D, const int32_t *q_len,
                               const int32_t *kv_len, int left, int right, int sinks, float scale, void *stream) {
    using namespace tpmd;
    auto fail = [](const char *m) { return tpk_fail(std::string("tpk_attn_window: ") + m); };
    constexpr int MAX_T = 1 << 30;
    if (dtype != TPMD_DTYPE_F32 && dtype != TPMD_DTYPE_F16) return fail("dtype");
    if (B < 0 || Tq < 0 || Tk < 0 || Tq > MAX_T || Tk > MAX_T || Hq < 0 || Hkv < 0 || D < 1 || D > 256)
        return fail("bad shape");
    if (Hkv > 0 ? Hq % Hkv != 0 : Hq != 0) return fail("Hq must be a multiple of Hkv");
    if (sinks < 0) return fail("sinks must not be negative");
    if (!(scale - scale == 0.0f)) return fail("scale must be finite");
    if (B == 0 || Tq == 0 || Hq == 0) return 0;  // no rows: nothing to write (pointers may be NULL)
    if (!strides || !q || !out || (Tk > 0 && (!k || !v))) return fail("null pointer");
    if (((uintptr_t) q | (uintptr_t) k | (uintptr_t) v | (uintptr_t) out) & (dtype == TPMD_DTYPE_F16 ? 1 : 3) ||
        ((uintptr_t) q_len | (uintptr_t) kv_len) & 3)
        return fail("a pointer is not aligned to its element type");
    if (!own_rows(strides + 9, B, Tq, Hq, D)) return fail("output rows overlap");
    attn_desc d{};
    d.q = q;
    d.k = k;
    d.v = v;
    d.out = out;
    for (int i = 0; i < 3; i++) {
        d.qs[i] = strides[i];
        d.ks[i] = strides[3 + i];
        d.vs[i] = strides[6 + i];
        d.os[i] = strides[9 + i];
    }
    d.f16 = dtype == TPMD_DTYPE_F16;
    d.B = B;
    d.Tq = Tq;
    d.Tk = Tk;
    d.Hq = Hq;
    d.Hkv = Hkv;
    d.D = D;
    d.q_len = q_len;
    d.kv_len = kv_len;
    d.left = left < 0 ? -1 : std::min(left, MAX_T);
    d.right = right < 0 ? -1 : std::min(right, MAX_T);
    d.sinks = std::min(sinks, MAX_T);
    d.scale = scale;
    const void *ptrs[] = {q, out, q_len, kv_len, Tk > 0 ? k : nullptr, Tk > 0 ? v : nullptr};
    tpk_device_scope dev(ptrs, 6);
    if (!dev.ok()) return fail(dev.why);
    const cudaError_t e = launch_attn(d, (cudaStream_t) stream);
    if (e == cudaErrorInvalidValue) return fail("too many rows, or the launch was refused");
    if (e != cudaSuccess) return fail(cudaGetErrorString(e));
    return 0;
}

extern "C" int tpk_attn_window_packed(const int64_t args[30]) {
    tpmd::packed_args p{args};
    const void *q = p.ptr(), *k = p.ptr(), *v = p.ptr();
    void *out = p.ptr();
    const int64_t *strides = p.a;
    p.a += 12;
    const int dtype = p.i32(), B = p.i32(), Tq = p.i32(), Tk = p.i32(), Hq = p.i32(), Hkv = p.i32(), D = p.i32();
    const int32_t *q_len = (const int32_t *) p.ptr(), *kv_len = (const int32_t *) p.ptr();
    const int left = p.i32(), right = p.i32(), sinks = p.i32();
    const float scale = (float) p.f64();
    void *stream = p.ptr();
    if (!p.fits) return tpmd::tpk_fail("tpk_attn_window: an argument is out of its range");
    return tpk_attn_window(q, k, v, out, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_len, kv_len, left, right, sinks,
                           scale, stream);
}
