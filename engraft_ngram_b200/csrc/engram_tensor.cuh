// engram_tensor.cuh -- what the tcgen05 kernels share: mbarriers with bounded
// waits, TMA tile loads (no multicast), MMA commits and tensor-map encoding; and
// how they and the kernels around them are launched.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "engram_common.cuh"

namespace engram {

constexpr long long kSpinLimit = 1ll << 24;  // polls of a barrier before a wait gives up

// Waits that gave up in this source file's kernels, where no counter was given (engram_waits_given_up adds the files').
static __device__ int g_waits_given_up;
inline int64_t read_given_up(const int& symbol) {
    int v = 0;
    return cudaMemcpyFromSymbol(&v, symbol, sizeof(v)) == cudaSuccess ? v : ENGRAM_ERR_CUDA;
}
int64_t gemm_waits_given_up();
int64_t adapter_waits_given_up();
int64_t ortho_waits_given_up();

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait for the phase with the given parity; false (and *err, or this file's own count, raised) on timeout.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int* err, long long limit = kSpinLimit) {
    for (long long it = 0; it < limit; it++)
        if (mbar_try_wait(bar, parity)) return true;
    atomicAdd(err ? err : &g_waits_given_up, 1);
    return false;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}

// ---- launches that overlap the one before them -----------------------------------

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

inline int64_t align256(int64_t b) { return (b + 255) & ~int64_t(255); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned_to(const void* p, int32_t dtype) {
    return ((uintptr_t)p & (dtype == ENGRAM_DTYPE_F32 ? 3u : 1u)) == 0;
}

template <typename... P, typename... A>
inline cudaError_t launch(void (*kernel)(P...), const cudaLaunchConfig_t& cfg, A... args) {
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Starts a kernel; after = true: it may start while the launch before it still runs (it waits for that
// one's results itself, griddepcontrol.wait), which hides the start and its first loads.
// MOST: the most dynamic shared memory a launch of the kernel takes (0: always `smem`).  CLUSTER: blocks along x
// of a cluster; a grid's third dimension of more than one is a cluster too.
template <auto KERNEL, int MOST = 0, int CLUSTER = 1, typename... A>
int start(dim3 grid, int threads, int smem, bool after, cudaStream_t st, A... args) {
    if (smem > 48 * 1024 || MOST > 48 * 1024) {
        static bool allowed[64] = {false};
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !allowed[dev]) {
            if (cudaFuncSetAttribute((const void*)KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     MOST ? MOST : smem) != cudaSuccess)
                return ENGRAM_ERR_CUDA;
            if (dev >= 0 && dev < 64) allowed[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    if (after) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (CLUSTER > 1 || grid.z > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs++].val.clusterDim = {CLUSTER, 1, CLUSTER > 1 ? 1 : grid.z};
    }
    cfg.attrs = attr;
    const cudaError_t e = launch(KERNEL, cfg, args...);
    count_launches(1);
    return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? ENGRAM_OK : ENGRAM_ERR_CUDA;
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

}  // namespace engram
