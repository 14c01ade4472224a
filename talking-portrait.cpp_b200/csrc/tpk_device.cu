// Device selection and the expired-wait word of the enqueue-only op entry
// points (tpk_gemm_f8, tpk_attn_window, tpk_quant_f8; include/tpmd.h).
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/tpmd.h"
#include "tpmd_internal.h"

namespace tpmd {
namespace {
// one per device (each device loads its own copy of the module)
__device__ int g_tpk_expired;
}  // namespace

tpk_device_scope::tpk_device_scope(const void *const *ptrs, int n) {
    for (int i = 0; i < n; i++) {
        if (!ptrs[i]) continue;
        cudaPointerAttributes a{};
        if (cudaPointerGetAttributes(&a, ptrs[i]) != cudaSuccess) {
            cudaGetLastError();
            why = "no CUDA device, or a pointer that CUDA does not know";
            return;
        }
        if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
            why = "a pointer is not device memory";
            return;
        }
        if (device >= 0 && a.device != device) {
            why = "the pointers lie on several devices";
            return;
        }
        device = a.device;
    }
    int cur = -1;
    if (device < 0 || cudaGetDevice(&cur) != cudaSuccess) {
        cudaGetLastError();
        why = "no CUDA device";
        return;
    }
    if (cur == device) return;
    if (cudaSetDevice(device) != cudaSuccess) {
        cudaGetLastError();
        why = "cudaSetDevice failed";
        return;
    }
    prev_ = cur;
}

tpk_device_scope::~tpk_device_scope() {
    if (prev_ >= 0) cudaSetDevice(prev_);
}

int *tpk_err_word() {
    static std::mutex mu;
    static int *word[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    std::lock_guard<std::mutex> g(mu);
    if (!word[dev]) {
        void *p = nullptr;
        if (cudaGetSymbolAddress(&p, g_tpk_expired) != cudaSuccess) return nullptr;
        word[dev] = (int *) p;
    }
    return word[dev];
}

}  // namespace tpmd

extern "C" int tpk_device_status(void *stream) {
    using namespace tpmd;
    cudaError_t e = cudaStreamSynchronize((cudaStream_t) stream);
    int flag = 0;
    int *w = e == cudaSuccess ? tpk_err_word() : nullptr;
    if (e == cudaSuccess && !w) e = cudaErrorUnknown;
    // on the caller's stream: a legacy-stream copy would wait for every other one
    if (e == cudaSuccess) e = cudaMemcpyAsync(&flag, w, sizeof flag, cudaMemcpyDeviceToHost, (cudaStream_t) stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t) stream);
    if (e == cudaSuccess && flag) e = cudaMemsetAsync(w, 0, sizeof(int), (cudaStream_t) stream);
    if (e == cudaSuccess && flag) e = cudaStreamSynchronize((cudaStream_t) stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return tpk_fail(std::string("tpk_device_status: ") + cudaGetErrorString(e));
    }
    return flag ? tpk_fail("a pipeline wait timed out (results invalid)") : 0;
}
