// Kernel launches of the token layers.
#pragma once

#include "common.cuh"

namespace bou {

struct LaunchShape {
    dim3 grid;
    int threads;
    size_t smem = 0;
    int cluster = 1;
    // The launch directly before this one on the stream is ours and lets this
    // one start early: the kernel calls wait_for_previous() before it touches
    // what the previous one reads or writes.
    bool chained = false;
};

template <typename Kernel, typename... Args>
int launch_kernel(const BulletOuCudaCppContext* ctx, const char* label, Kernel kernel, const LaunchShape& shape, Args... args) {
    if (shape.smem > 48 * 1024) {
        const cudaError_t st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shape.smem));
        if (st != cudaSuccess) return fail(label, st);
    }
    cudaLaunchConfig_t config{};
    config.gridDim = shape.grid;
    config.blockDim = dim3(shape.threads);
    config.dynamicSmemBytes = shape.smem;
    config.stream = ctx->stream;
    cudaLaunchAttribute attrs[2];
    config.attrs = attrs;
    if (shape.cluster > 1) {
        attrs[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[config.numAttrs++].val.clusterDim = {static_cast<unsigned>(shape.cluster), 1, 1};
    }
    if (shape.chained) {
        attrs[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    const cudaError_t st = cudaLaunchKernelEx(&config, kernel, args...);
    return st != cudaSuccess ? fail(label, st) : 0;
}

// Everything of the previous kernel is done and visible (at once where the
// launch was not chained).
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// A chained next kernel may be set up on the SMs that have room.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }

}  // namespace bou
