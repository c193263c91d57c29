// ============================================================================
//  launch.cuh -- launch bookkeeping shared by every kernel file.
// ============================================================================
#pragma once

#include "common.cuh"

namespace tg {

void count_launch(const char* name);  // one per kernel launch (tg_kernel_launch_count, tg_last_kernel_name)
void require_device();   // throws TG_ERR_NO_DEVICE without a GPU

// Lets `kernel` be launched with up to `most` bytes of dynamic shared memory: the
// most that any call of it needs, since a limit that followed each call's own need
// could be lowered by another host thread between this thread's setting and launch.
template <class K>
inline void allow_shared(K kernel, int most) {
    TG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
}
constexpr int kMaxShared = 227 * 1024;  // of a block, its static shared memory included

// Launch `kernel<<<grid, block, smem, stream>>>(args...)`, count it and check
// the launch.  Empty grids launch nothing.
template <class K, class... A>
inline void launch(const char* name, K kernel, dim3 grid, dim3 block, size_t smem,
                   cudaStream_t s, A... args) {
    if (grid.x == 0 || grid.y == 0 || grid.z == 0) return;
    kernel<<<grid, block, smem, s>>>(args...);
    count_launch(name);
    TG_LAUNCH_CHECK(name);
}

// The same with programmatic dependent launch: the kernel's blocks may start
// while the stream's previous kernel still runs, and must call
// wait_for_previous() before they read or write memory.  Launch latency and a
// kernel's own set-up then overlap with its predecessor's last blocks.
template <class K, class... A>
inline void launch_dependent(const char* name, K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t s, A... args) {
    if (grid.x == 0 || grid.y == 0 || grid.z == 0) return;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), name);
    count_launch(name);
}

#ifdef __CUDACC__
// Every kernel launched that way: lets the next one start early, and returns
// once the previous one is complete and its writes are visible.
__device__ __forceinline__ void wait_for_previous() {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}
#endif

// Common argument checks with the reference's wording.
inline void check_ld(const char* fn, const char* what, int64_t ld, int64_t cols) {
    if (ld < cols)
        invalid(std::string(fn) + ": leading dimension of " + what + " (" + std::to_string(ld) +
                ") is smaller than its column count (" + std::to_string(cols) + ")");
}

inline void check_ptr(const char* fn, const char* what, const void* p, bool needed) {
    if (needed && p == nullptr) invalid(std::string(fn) + ": " + what + " is NULL");
}

}  // namespace tg
