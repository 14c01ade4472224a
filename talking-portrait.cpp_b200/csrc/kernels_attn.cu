// Sliding-window attention with first tokens that stay visible
// (tpk_attn_window, include/tpmd.h), on the CUDA cores: any strides,
// alignment and type.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max),
//   over keys j < min(L, p + right + 1) with j >= p - left or j < sinks,
//   p = L - n + i
//
// One warp per query row and head; the visible keys are the two ranges
// [0, sinks) and [p - left, p + right], walked with a running maximum and
// sum (f32), so keys outside them are never read.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "../../include/tpmd.h"
#include "attn_row.cuh"
#include "tpmd_internal.h"

namespace tpmd {
namespace {

template <typename T, int EPL>
__global__ void __launch_bounds__(128) attn_row_kernel(const __grid_constant__ attn_desc p, int64_t rows) {
    const int lane = threadIdx.x & 31;
    const int64_t g = ((int64_t) blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (g >= rows) return;
    const int i = (int) (g % p.Tq), h = (int) (g / p.Tq % p.Hq), b = (int) (g / p.Tq / p.Hq);
    const int n = p.q_len ? min(max(p.q_len[b], 0), p.Tq) : p.Tq;
    const int L = p.kv_len ? min(max(p.kv_len[b], 0), p.Tk) : p.Tk;
    if (i < n) attn_row<T, EPL>(p, b, h, i, n, L, lane);
}

template <typename T>
cudaError_t run_rows(const attn_desc &d, cudaStream_t st) {
    const int64_t rows = (int64_t) d.B * d.Hq * d.Tq, blocks = (rows + 3) / 4;
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    if (d.D <= 64) attn_row_kernel<T, 2><<<(unsigned) blocks, 128, 0, st>>>(d, rows);
    else if (d.D <= 128) attn_row_kernel<T, 4><<<(unsigned) blocks, 128, 0, st>>>(d, rows);
    else attn_row_kernel<T, 8><<<(unsigned) blocks, 128, 0, st>>>(d, rows);
    return cudaGetLastError();
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

cudaError_t launch_attn_simt(const attn_desc &d, cudaStream_t st) {
    return d.f16 ? run_rows<__half>(d, st) : run_rows<float>(d, st);
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
    const cudaError_t e = attn_tc_supported(d) ? launch_attn_tc(d, (cudaStream_t) stream) : launch_attn_simt(d, (cudaStream_t) stream);
    if (e == cudaErrorInvalidValue) return fail("too many rows, or the launch was refused");
    if (e != cudaSuccess) return fail(cudaGetErrorString(e));
    return 0;
}
