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
// A CTA has 16 RPT rows (tokens times the query heads of a group, so that
// these share a key head's tiles) and goes through the keys that any of them
// sees, 32 at a time, with a running maximum and sum: one list of the sinks
// and the window behind them. K and V tiles come by cp.async, one ahead.
// Thread (rg, kx) = (tid / 8, tid % 8) has rows rg + 16 j: their scores with
// keys kx + 8 i, then columns 4 kx + 32 i of their outputs (register tiles
// of 4 x 4 RPT: the FMAs need one 16-byte shared load for every eight).
// Where the rows do not fill the SMs, a cluster of up to eight CTAs shares
// the tiles out and joins its parts in shared memory in a fixed order.
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

template <int DC, int RPT>
struct tile_cfg {
    static constexpr int BM = 16 * RPT, KT = 32, DP = 32 * DC, LD = DP + 4, PLD = KT + 4;
    static constexpr int KV = KT * LD;  // floats a K or V tile
    static constexpr int SMEM = (BM * LD + 4 * KV + BM * PLD + 2 * BM) * 4;
    static_assert(BM * LD <= 4 * KV, "a part fits the tiles");
    static_assert(SMEM <= 232448, "shared memory");
};

template <typename T, int DC, int RPT>
__global__ void __launch_bounds__(128)
attn_tile_kernel(const __grid_constant__ tile_params p) {
    using cfg = tile_cfg<DC, RPT>;
    constexpr int KT = cfg::KT, LD = cfg::LD;
    extern __shared__ float4 smem4[];
    float *sq = (float *) smem4, *skv = sq + cfg::BM * LD, *sp = skv + 4 * cfg::KV;
    float2 *s_ml = (float2 *) (sp + cfg::BM * cfg::PLD);
    const attn_desc &d = p.d;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, kx = tid % 8, rg = tid / 8;
    int idx = blockIdx.x;
    const int rank = idx % p.splits;
    idx /= p.splits;
    const int bh = idx % (d.B * d.Hkv), qt = p.qtiles - 1 - idx / (d.B * d.Hkv);  // (the last rows see most keys)
    const int b = bh / d.Hkv, hk = bh % d.Hkv;
    const int n = d.q_len ? min(max(__ldg(d.q_len + b), 0), d.Tq) : d.Tq;
    const int L = d.kv_len ? min(max(__ldg(d.kv_len + b), 0), d.Tk) : d.Tk;
    const int64_t r0 = (int64_t) qt * cfg::BM;  // rows: token g + head of the group
    const int rows = (int) min((int64_t) cfg::BM, (int64_t) n * p.g - r0);
    if (rows <= 0) return;  // (the whole cluster alike)
    const int64_t base = (int64_t) L - n;
    const key_range kr = keys_of(d, L, base + r0 / p.g, base + (r0 + rows - 1) / p.g);
    // the keys that some row sees, in one list: the sinks, then the window
    const int keys = kr.first + kr.hi - kr.lo, nall = (keys + KT - 1) / KT;
    auto key_at = [&](int i) { return i < kr.first ? i : i - kr.first + kr.lo; };
    const int i0 = (int) ((int64_t) nall * rank / p.splits), i1 = (int) ((int64_t) nall * (rank + 1) / p.splits);
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
    // tile i of the list into buffer i & 1, zeros behind its end
    auto load = [&](int i) {
        float *k = skv + (i & 1) * 2 * cfg::KV, *v = k + cfg::KV;
        for (int e = tid; e < KT * DC * 8; e += 128) {
            const int r = e / (DC * 8), x = e % (DC * 8) * 4, left = i * KT + r < keys ? d.D - x : 0;
            const int64_t key = key_at(i * KT + r);
            const T *ks = kbase + key * d.ks[1] + x, *vs = vbase + key * d.vs[1] + x;
            if (sizeof(T) == 4 && p.kv_vec && (left >= 4 || left <= 0)) {
                const int bytes = left > 0 ? 16 : 0;  // 0: zeros, nothing is read
                if (!bytes) {
                    ks = kbase;
                    vs = vbase;
                }
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(k + r * LD + x)), "l"(ks),
                             "r"(bytes)
                             : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(v + r * LD + x)), "l"(vs),
                             "r"(bytes)
                             : "memory");
            } else {
                *reinterpret_cast<float4 *>(k + r * LD + x) = load4(ks, left, p.kv_vec);
                *reinterpret_cast<float4 *>(v + r * LD + x) = load4(vs, left, p.kv_vec);
            }
        }
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
    if (i0 < i1) load(i0);
    for (int i = i0; i < i1; i++) {
        if (i + 1 < i1) {
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
    // parts to shared memory (in the tiles' place), then a row at a time to
    // a warp: the sum over the cluster's parts, and out
#pragma unroll
    for (int j = 0; j < RPT; j++) {
#pragma unroll
        for (int w = 4; w > 0; w >>= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], w);
        const int r = rg + 16 * j;
        if (kx == 0) s_ml[r] = make_float2(m[j], l[j]);
#pragma unroll
        for (int x = 0; x < DC; x++) *reinterpret_cast<float4 *>(skv + r * LD + 4 * kx + 32 * x) = o[j][x];
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    const int lane = tid & 31, warp = tid >> 5;
    for (int r = rank * 4 + warp; r < rows; r += p.splits * 4) {
        float M = -INFINITY, sl = 0.0f, v[DC];
        for (int k = 0; k < p.splits; k++) M = fmaxf(M, ld_part(&s_ml[r].x, k, p.splits));
#pragma unroll
        for (int x = 0; x < DC; x++) v[x] = 0.0f;
        for (int k = 0; k < p.splits; k++) {
            const float mk = ld_part(&s_ml[r].x, k, p.splits), lk = ld_part(&s_ml[r].y, k, p.splits);
            const float f = mk == -INFINITY ? lk : exp2f(mk - M);  // (a part that saw no key: 0; NaN stays)
            sl = fmaf(f, lk, sl);
#pragma unroll
            for (int x = 0; x < DC; x++) v[x] = fmaf(f, ld_part(skv + r * LD + lane + 32 * x, k, p.splits), v[x]);
        }
        const int tok = (int) ((r0 + r) / p.g), h = hk * p.g + (int) ((r0 + r) % p.g);
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
    if (p.splits > 1) cluster_sync_all();  // no CTA leaves while others read its parts
}

template <typename T, int DC, int RPT>
cudaError_t run_tile(tile_params &p, cudaStream_t st) {
    using cfg = tile_cfg<DC, RPT>;
    const attn_desc &d = p.d;
    const int64_t rows = (int64_t) d.Tq * p.g, qtiles = (rows + cfg::BM - 1) / cfg::BM, bh = (int64_t) d.B * d.Hkv;
    // the keys that a tile of rows can see, in tiles
    int64_t keys = d.Tk;
    if (d.left >= 0 && d.right >= 0)
        keys = std::min<int64_t>(keys, cfg::BM / p.g + 2 + (int64_t) d.left + d.right + d.sinks);
    if (qtiles > INT32_MAX || bh * qtiles > INT32_MAX / 8) return cudaErrorInvalidValue;
    p.qtiles = (int) qtiles;
    p.splits = cluster_size(bh * qtiles, (keys + 63) / 64);  // parts down to two tiles of keys
    static std::mutex mu;
    static uint64_t attr_set = 0;  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> g(mu);
        if (!(attr_set >> (dev & 63) & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(attn_tile_kernel<T, DC, RPT>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, cfg::SMEM);
            if (e != cudaSuccess) return e;
            attr_set |= 1ull << (dev & 63);
        }
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned) (bh * qtiles * p.splits), 1, 1);
    lc.blockDim = dim3(128, 1, 1);
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
    const cudaError_t e = cudaLaunchKernelEx(&lc, attn_tile_kernel<T, DC, RPT>, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int DC>
cudaError_t run_rows(tile_params &p, cudaStream_t st) {
    // 64 rows a CTA (32 of wide heads) where that fills the SMs, else 16
    constexpr int RPT = DC > 4 ? 2 : 4;
    const int64_t rows = (int64_t) p.d.Tq * p.g;
    if ((rows + 16 * RPT - 1) / (16 * RPT) * p.d.B * p.d.Hkv >= sm_count()) return run_tile<T, DC, RPT>(p, st);
    return run_tile<T, DC, 1>(p, st);
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
