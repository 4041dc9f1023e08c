// Host-side plumbing shared by the translation units of libdfb_cuda: the error record behind
// dfb_last_error(), CUDA-call checks and kernel launches.
#pragma once
#include <cuda_runtime.h>

#include "../../../include/diffuse_b200.h"

namespace dfb {

// Records the message for dfb_last_error() (thread-local) and returns code.
int set_err(int code, const char *fmt, ...);

#define CK(call)                                                                                   \
    do {                                                                                           \
        cudaError_t e_ = (call);                                                                   \
        if (e_ != cudaSuccess) {                                                                   \
            cudaGetLastError(); /* else the next launch's check finds it */                        \
            return set_err(e_ == cudaErrorMemoryAllocation ? DFB_ERR_NOMEM : DFB_ERR_CUDA,         \
                           "%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); \
        }                                                                                          \
    } while (0)
#define RET(x)                 \
    do {                       \
        int r_ = (x);          \
        if (r_ != DFB_OK) return r_; \
    } while (0)

// Programmatic dependent launch: a kernel launched this way may start while the
// previous kernel of the stream is finishing; every such kernel executes
// griddepcontrol.wait before it touches memory the previous kernels write.
// DIFFUSE_PDL=0 turns it off (plain stream order).
bool pdl_enabled();

template <typename... KArgs, typename... Args>
static cudaError_t launch_k(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl,
                            Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = (pdl && pdl_enabled()) ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace dfb
