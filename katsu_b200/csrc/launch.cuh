// Launches whose start overlaps the end of the kernel in front of them on the stream (programmatic dependent launch).
//
// A kernel launched this way may be resident while its predecessor still runs: before it touches global memory that the
// predecessor (or anything before it) reads or writes it must call launch_wait(), which returns once all of that is
// complete and visible.  launch_next(), called by every block, lets the successor start; called early it hides the
// successor's launch and prologue.  In a chain of small kernels those were most of the time (a 14 x 14 layer's forward:
// three kernels, 23 us).
#pragma once

#include <string.h>

#include "common.cuh"

__device__ __forceinline__ void launch_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Once per kernel and device (and whenever more is asked for): its dynamic shared memory, and the largest shared-memory
// partition of the SM, so that kernels that follow each other do not make the SM re-partition its memory, which it only
// does when it is idle.  Kernels that live on loads in flight are better off without (largest = false): these take L1, which
// that partition leaves 28 KiB (a step over 1.2 GB of gradients and weights each: 682 us with it, 506 without).
int32_t katsu_prepare_kernel(katsu_cuda_ctx *ctx, const void *kernel, size_t smem, bool largest = true);

// early: the launch may start under its predecessor's end.  Only for grids whose blocks the device holds all at once: one that is
// handed out in waves is launched plainly, and its blocks do not call launch_next().  (One early form in waves hung; why, is not
// known.)  Blocks are counted for a device without other work.  Beside a predecessor fewer fit at first, and the rest come as its
// blocks end: these are all running by then, or nothing would start early, and wait for nothing that comes later.
template <typename... Params, typename... Args>
int32_t katsu_launch(katsu_cuda_ctx *ctx, bool early, void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem,
                     unsigned cluster, Args &&...args) {
    cudaLaunchConfig_t config;
    memset(&config, 0, sizeof(config));
    config.gridDim = dim3(grid, 1, 1);
    config.blockDim = dim3(block, 1, 1);
    config.dynamicSmemBytes = smem;
    config.stream = ctx->stream;
    cudaLaunchAttribute attributes[2];
    memset(attributes, 0, sizeof(attributes));
    config.attrs = attributes;
    if (early) {
        attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[0].val.programmaticStreamSerializationAllowed = 1;
        config.numAttrs = 1;
    }
    if (cluster > 1) {
        cudaLaunchAttribute &of_cluster = attributes[config.numAttrs++];
        of_cluster.id = cudaLaunchAttributeClusterDimension;
        of_cluster.val.clusterDim.x = cluster;
        of_cluster.val.clusterDim.y = of_cluster.val.clusterDim.z = 1;
    }
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
    ctx->launches += 1;
    if (err != cudaSuccess) {
        cudaGetLastError();
        return katsu_set_error(KATSU_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(err));
    }
    return KATSU_OK;
}

template <typename... Params, typename... Args>
int32_t katsu_launch_chained(katsu_cuda_ctx *ctx, void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem,
                             unsigned cluster, Args &&...args) {
    return katsu_launch(ctx, true, kernel, grid, block, smem, cluster, static_cast<Args &&>(args)...);
}
