// jq_host.cuh -- what the library's translation units share: error returns,
// and launches that overlap the previous kernel's end.
#pragma once
#include <cuda_runtime.h>

#include "../../include/jq.h"

namespace jq {

int fail(int code, const char *msg);                  // sets jq_last_error(), returns code
int cuda_fail(cudaError_t err, const char *where);    // as fail, JQ_ERR_CUDA
int device_sms(int &sms);                             // SMs of the current device

#define CU(call)                                                    \
    do {                                                            \
        cudaError_t _e = (call);                                    \
        if (_e != cudaSuccess) return cuda_fail(_e, #call);         \
    } while (0)

// Entry of the kernels launched with programmatic dependent launch
// (launch_pdl): let the next kernel in the stream be scheduled early, then
// wait until the previous one has completed and its writes are visible,
// before the first access to caller memory.
__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Programmatic dependent launch: the kernel may be scheduled while the
// previous kernel in the stream drains (the rules kernel's slowest envs, the
// observation kernel's last units), load its board tables into shared
// memory, then wait (griddepcontrol.wait) for that kernel to complete
// before touching any state.  Kernels launched this way call
// griddepcontrol.wait before their first access to caller memory.
template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                              Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace jq
