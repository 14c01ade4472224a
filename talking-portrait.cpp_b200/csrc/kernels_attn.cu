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
// head's tiles. A CTA has up to 16; the keys that any of them sees are one
// list, the sinks and the window behind them. Every warp has all the rows and
// its own share of that list, in tiles of 8 keys with a running maximum and
// sum, K and V by cp.async two tiles ahead, and waits for nothing but its
// copies. Lane (rg, kx) = (lane / 8, lane % 8) holds columns 4 kx + 32 i of
// rows rg + 4 j and of their outputs in registers: eight lanes sum a row's
// scores over their columns, key kx's to lane kx, and each 16-byte shared
// load of K or V feeds R rows. The warps' parts join in shared memory; where
// CTAs do not fill the SMs a cluster of up to eight shares the list and joins
// over distributed shared memory; always in the same order.
//
// Measured, f32: 16 sequences of one token over 4100 keys, 16 heads of 128 on
// 4 (269 MB): 57 us, 4.7 TB/s (latency of the shared loads with eight warps an
// SM; tiles of 64 rows with all threads in step took 241 us). 4096 tokens, 16
// heads of 128 on 4, 1024 keys each: 1.03 ms, 29 TFLOP/s of what the mask
// leaves, the multiply-add pipe busy half of the time (the same eight warps:
// registers; tiles of 64 rows 0.91 ms, but 173 us against 120 at 3000 tokens
// of 8 heads, 200 keys, where whole tiles of 64 do not share out evenly). The
// sampler's 60 frames of 3 x 8 heads over 5 + 10 keys: 9.4 us, 96 CTAs that
// wait for their loads.
// f16 here has no copies ahead of its use, a load at a time: 2000 tokens, 8
// heads on 2, 512 keys each, 1.9 ms in heads of 160 or 256 (16 us in heads of
// 128 on the tensor cores); 16 tokens over 4100 keys, 8 heads of 256 on 2,
// 0.56 ms; heads of 128 in rows off 16-byte boundaries 0.40 ms.
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
#include "tc_ops.cuh"
#include "tpmd_internal.h"

namespace tpmd {
namespace {

struct rows_params {
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
__device__ __forceinline__ void store_row(const rows_params &p, int b, int hk, int64_t row, int n, int L, float sl,
                                          const float (&v)[DC], int lane) {
    const attn_desc &d = p.d;
    const int tok = (int) ((uint32_t) row / (uint32_t) p.g), h = hk * p.g + (int) ((uint32_t) row - tok * (uint32_t) p.g);
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

template <int DC, int R, int WARPS>
struct row_cfg {
    static constexpr int KT = 8, BM = 4 * R, LD = 32 * DC + 4, PLD = KT + 4;
    static constexpr int KV = KT * LD;                  // floats a K or V tile
    static constexpr int WARP = 4 * KV + BM * PLD;      // floats a warp: two tiles of each, weights
    static constexpr int SMEM = (WARPS * WARP + 2 * WARPS * BM) * 4;
    static_assert(BM <= 4 * KT, "a part fits the tiles");
    static_assert(SMEM <= 232448, "shared memory");
};

// 4 R rows, all by each of the CTA's warps, which share the keys out and run
// on their own until they join
template <typename T, int DC, int R, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
attn_rows_kernel(const __grid_constant__ rows_params p) {
    using cfg = row_cfg<DC, R, WARPS>;
    constexpr int KT = cfg::KT, LD = cfg::LD, BM = cfg::BM;
    extern __shared__ float4 smem4[];
    const attn_desc &d = p.d;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kx = lane % 8, rg = lane / 8;
    float *parts = (float *) smem4, *skv = parts + warp * cfg::WARP, *sp = skv + 4 * cfg::KV;
    float2 *s_ml = (float2 *) (parts + WARPS * cfg::WARP);
    int idx = blockIdx.x;
    const int rank = idx % p.splits;
    idx /= p.splits;
    const int bh = idx % (d.B * d.Hkv), qt = p.qtiles - 1 - idx / (d.B * d.Hkv);
    const int b = bh / d.Hkv, hk = bh % d.Hkv;
    const int n = d.q_len ? min(max(d.q_len[b], 0), d.Tq) : d.Tq;
    const int L = d.kv_len ? min(max(d.kv_len[b], 0), d.Tk) : d.Tk;
    const int64_t r0 = (int64_t) qt * BM;
    const int rows = (int) min((int64_t) BM, (int64_t) n * p.g - r0);
    if (rows <= 0) return;  // (the whole cluster alike)
    const int64_t base = (int64_t) L - n;
    const key_range kr = keys_of(d, L, base + (uint32_t) r0 / (uint32_t) p.g, base + (uint32_t) (r0 + rows - 1) / (uint32_t) p.g);
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
    key_range kk[R];
    float m[R], l[R];
    uint64_t q[R][DC][2], o[R][DC][2];  // columns 4 kx + 32 i of the rows, in pairs
#pragma unroll
    for (int j = 0; j < R; j++) {
        // (rows fit 32 bits: launch)
        const uint32_t r = (uint32_t) r0 + min(rg + 4 * j, rows - 1), tok = r / (uint32_t) p.g, h = r - tok * p.g;
        const int64_t pos = base + tok;
        kk[j] = keys_of(d, L, pos, pos);
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const int x = 4 * kx + 32 * i;
            const float4 f = load4((const T *) d.q + b * d.qs[0] + tok * d.qs[1] + (hk * p.g + h) * d.qs[2] + x,
                                   d.D - x, p.q_vec);
            q[j][i][0] = pack2(f.x * p.c, f.y * p.c);
            q[j][i][1] = pack2(f.z * p.c, f.w * p.c);
            o[j][i][0] = o[j][i][1] = 0;
        }
    }
    for (int i = i0; i < i1; i++) {
        const float *k = skv + (i & 1) * cfg::KV, *v = skv + (2 + (i & 1)) * cfg::KV;
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        __syncwarp();
        const int here = min(KT, keys - i * KT);  // keys of the tile
        float s[R][KT];  // of the lane's columns
#pragma unroll
        for (int e = 0; e < KT; e++) {
            uint64_t s2[R];
#pragma unroll
            for (int j = 0; j < R; j++) s2[j] = 0;
#pragma unroll
            for (int x = 0; x < DC; x++) {
                const ulonglong2 kv = *reinterpret_cast<const ulonglong2 *>(k + e * LD + 4 * kx + 32 * x);
#pragma unroll
                for (int j = 0; j < R; j++) s2[j] = fma2(q[j][x][1], kv.y, fma2(q[j][x][0], kv.x, s2[j]));
            }
#pragma unroll
            for (int j = 0; j < R; j++) {
                const float2 h = unpack2(s2[j]);
                s[j][e] = h.x + h.y;
            }
        }
        __syncwarp();  // (K's buffer is loaded again)
        load_k(i + 2);
#pragma unroll
        for (int j = 0; j < R; j++) {
            // the eight lanes' sums, key kx's to lane kx
#pragma unroll
            for (int w = 4; w > 0; w >>= 1)
#pragma unroll
                for (int e = 0; e < w; e++) {
                    const float mine = kx & w ? s[j][e + w] : s[j][e], other = kx & w ? s[j][e] : s[j][e + w];
                    s[j][e] = mine + __shfl_xor_sync(0xffffffffu, other, w);
                }
            const int key = key_at(i * KT + kx);
            const bool sees = kx < here && key < kk[j].hi && (key >= kk[j].lo || key < d.sinks);
            const float sc = sees ? s[j][0] : -INFINITY;
            float mn = fmaxf(m[j], sc);
#pragma unroll
            for (int w = 4; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
            const float zero = mn == -INFINITY ? 0.0f : mn, f = exp2f(m[j] - zero), w = exp2f(sc - zero);
            m[j] = mn;
            l[j] = fmaf(l[j], f, w);
            sp[(rg + 4 * j) * cfg::PLD + kx] = w;
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
cudaError_t launch(rows_params &p, int rows, int threads, int smem, int64_t most_splits, cudaStream_t st) {
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
cudaError_t run_warps(rows_params &p, cudaStream_t st) {
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
cudaError_t run_few(rows_params &p, cudaStream_t st) {
    // eight warps a CTA hide more of each other's latency; with four, two or
    // three CTAs fit an SM and one's start and end hide behind the others
    // (768 rows of 128 over 200 keys each: four warps 39 us, eight 68; four
    // rows over 4100 keys, 64 times: 71, 58)
    const int64_t ctas = ((int64_t) p.d.Tq * p.g + 4 * R - 1) / (4 * R) * p.d.B * p.d.Hkv;
    if (DC > 4 || ctas >= 2 * sm_count()) return run_warps<T, DC, R, 4>(p, st);
    return run_warps<T, DC, R, (DC > 4 ? 4 : 8)>(p, st);
}

template <typename T, int DC>
cudaError_t run_rows(rows_params &p, cudaStream_t st) {
    constexpr int MOST = DC > 4 ? 2 : 4;  // (of wide heads eight rows: registers)
    const int64_t rows = (int64_t) p.d.Tq * p.g;
    return rows <= 4 ? run_few<T, DC, 1>(p, st) : rows <= 8 ? run_few<T, DC, 2>(p, st) : run_few<T, DC, MOST>(p, st);
}

template <typename T>
cudaError_t run_simt(const attn_desc &d, cudaStream_t st) {
    rows_params p{};
    p.d = d;
    p.g = d.Hq / d.Hkv;
    p.c = d.scale * 1.4426950408889634f;
    auto vec = [&](const void *x, const int64_t *s, int64_t n1, int64_t n2) {
        return !((uintptr_t) x & (4 * sizeof(T) - 1)) && (d.B == 1 || s[0] % 4 == 0) && (n1 <= 1 || s[1] % 4 == 0) &&
               (n2 <= 1 || s[2] % 4 == 0);
    };
    p.q_vec = vec(d.q, d.qs, d.Tq, d.Hq);
    p.kv_vec = vec(d.k, d.ks, d.Tk, d.Hkv) && vec(d.v, d.vs, d.Tk, d.Hkv);
    if (d.D <= 32) return run_rows<T, 1>(p, st);
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
