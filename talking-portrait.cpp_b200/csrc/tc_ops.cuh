// Building blocks of the 8-bit product, the quantiser and windowed attention,
// beside tc_ptx.cuh, which the convolutions share: their recorded DRAM traffic
// is keyed by that file's bytes.
#pragma once
#include "tc_ptx.cuh"

namespace tpmd {
namespace {

__device__ __forceinline__ void prefetch_map(const CUtensorMap *tm) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t) tm) : "memory");
}
// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e != 0;
}
// a bounded wait of a whole warp, one answer for all lanes
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
// both of two barriers' phases (their latencies overlap)
__device__ __forceinline__ bool warp_wait2(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1) {
    const bool r0 = mbar_try(bar0, parity0), r1 = mbar_try(bar1, parity1);
    if (__all_sync(0xffffffffu, r0 && r1)) return true;
    return warp_wait(bar0, parity0) && warp_wait(bar1, parity1);
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

// CTAs a cluster when n clusters share work out, at most `most`, for kernels
// with one CTA an SM: all n have to run at once. A cluster lies within a GPC
// (16 to 18 SMs), so pairs use every SM, clusters of four 128 or so, and one
// of eight a GPC is safe; sizes that do not divide a GPC's SMs leave some
// idle. (In 8 bits, 180x1024x4096: 16 clusters of eight 17.9 us, of four 9.9;
// 48 clusters of three 13.6 us, of two 8.4.)
inline int cluster_size(int64_t n, int64_t most) {
    if (most >= 8 && n <= 8) return 8;
    if (most >= 4 && n <= 32) return 4;
    return most >= 2 && 2 * n <= sm_count() ? 2 : 1;
}

}  // namespace
}  // namespace tpmd
