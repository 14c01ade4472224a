// What both forms of windowed attention share: the keys that rows see, and
// one query row by one warp, reading nothing but its visible keys, which a row
// that came out not finite is computed again with.
#pragma once
#include <cuda_fp16.h>

#include "tpmd_internal.h"

namespace tpmd {
namespace {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// two f32 in one register pair
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// the keys that a set of rows sees: [0, first) and [lo, hi), lo >= first
struct key_range {
    int first, lo, hi;
};
// of the rows at positions p0 .. p1
__device__ __forceinline__ key_range keys_of(const attn_desc &d, int L, int64_t p0, int64_t p1) {
    key_range k;
    k.hi = d.right < 0 ? L : (int) max((int64_t) 0, min((int64_t) L, p1 + d.right + 1));
    k.lo = d.left < 0 ? 0 : (int) min((int64_t) k.hi, max((int64_t) 0, p0 - d.left));
    k.first = min(d.sinks, k.lo);
    return k;
}

// row i of head h of sequence b, which has n rows and L keys; lane e holds
// columns e, e + 32, ... of the row (D <= 32 EPL)
template <typename T, int EPL>
__device__ __noinline__ void attn_row(const attn_desc &p, int b, int h, int i, int n, int L, int lane) {
    const int64_t pos = (int64_t) L - n + i;
    const int hi = (int) max((int64_t) 0, p.right < 0 ? (int64_t) L : min((int64_t) L, pos + p.right + 1));
    const int lo = p.left < 0 ? 0 : (int) min((int64_t) hi, max((int64_t) 0, pos - p.left));
    const int first = min(p.sinks, lo);
    const int hk = h / (p.Hq / p.Hkv);
    const T *q = (const T *) p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
    const T *kb = (const T *) p.k + b * p.ks[0] + hk * p.ks[2];
    const T *vb = (const T *) p.v + b * p.vs[0] + hk * p.vs[2];
    float qv[EPL], o[EPL];
#pragma unroll
    for (int e = 0; e < EPL; e++) {
        const int d = lane + 32 * e;
        qv[e] = d < p.D ? to_f(q[d]) * p.scale : 0.0f;
        o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int t = 0; t < first + hi - lo; t++) {
        const int64_t j = t < first ? t : t - first + lo;
        const T *k = kb + j * p.ks[1], *v = vb + j * p.vs[1];
        float s = 0.0f, vv[EPL];
#pragma unroll
        for (int e = 0; e < EPL; e++) {
            const int d = lane + 32 * e;
            s = fmaf(qv[e], d < p.D ? to_f(k[d]) : 0.0f, s);
            vv[e] = d < p.D ? to_f(v[d]) : 0.0f;
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;
        const float c = expf(m - base), w = expf(s - base);
        m = mn;
        l = l * c + w;
#pragma unroll
        for (int e = 0; e < EPL; e++) o[e] = fmaf(w, vv[e], o[e] * c);
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // NaN stays NaN
    T *out = (T *) p.out + b * p.os[0] + i * p.os[1] + h * p.os[2];
#pragma unroll
    for (int e = 0; e < EPL; e++) {
        const int d = lane + 32 * e;
        if (d < p.D) out[d] = from_f<T>(l == 0.0f ? 0.0f : o[e] * inv);
    }
}

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// *x of CTA `rank` of the cluster (its own shared memory where there is no cluster)
__device__ __forceinline__ float ld_part(const float *x, int rank, int ctas) {
    if (ctas == 1) return *x;
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t) __cvta_generic_to_shared(x)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

}  // namespace
}  // namespace tpmd
