// q8_launch.cuh — launches of the 8-bit row kernels, which follow one another
// closely (norm, product, cache), as programmatic dependents: a kernel's blocks
// may start while the last blocks of the one before it in the stream finish, and
// set up what touches no memory that those may still write or read; before_memory()
// then waits until they are done and their writes are visible. What such a kernel reads
// may thus be written while it already runs: its pointers must not promise otherwise
// (__restrict__, ld.global.nc, __ldg), or the compiler could read ahead of the wait.
// Grids of more than 64 blocks an SM start in the ordinary way. A norm (one block a row) and
// the product that follows it, in turn, took with no early start / this limit / early starts
// alone: 4096 rows of 4096 44.9 / 45.1 / 45.1 us, 8192 73.1 / 75.4 / 75.3, 12288 102.5 / 100.9 /
// 105.2, 32768 239 / 238 / 259, 65536 rows of 2048 210 / 208 / 230. The norm and its reading
// back: 2048 rows of 4096 17.6 / 17.2 / 17.2, 4096 34.0 / 33.0 / 33.0, 32768 215 / 215 / 213.
#pragma once
#include <cuda_runtime.h>

#include "jhq_common.h"

namespace jhq {

__device__ __forceinline__ void before_memory() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Once every block has called this (or ended), the next kernel's blocks may start.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... P, class... A>
void launch_q8(void (*kernel)(P...), dim3 grid, unsigned block, size_t smem, int cluster, cudaStream_t s, A... args) {
    constexpr int64_t MOST_EARLY = 148 * 64;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = (int64_t)grid.x * grid.y <= MOST_EARLY;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    JHQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

}  // namespace jhq
