// How the small ops are launched: with programmatic dependent launch.  Each lets its successor start at once and waits for its
// predecessor before it touches an operand, so that in a chain of op calls the next kernel's launch and set-up overlap the
// previous kernel's tail (worth 1-2 us per launch where a kernel itself takes 2 us).
#pragma once

#include "common.cuh"

namespace ib {

__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... KArgs, typename... Args>
static int32_t launch_op(ib_ctx *ctx, cudaStream_t s, void (*kernel)(KArgs...), uint32_t grid, uint32_t block, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    IB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, (KArgs)args...));
    ctx->launches++;
    return IB_OK;
}

}  // namespace ib
