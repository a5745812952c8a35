// pdl_launch.cuh -- launches of the small kernels with programmatic stream
// serialisation.
//
// A kernel launched this way may be resident before the kernels before it
// have finished, and its SM's L1 may then hold lines that they go on to
// change.  The kernels of several drafted tokens therefore read what an
// earlier kernel may have written past L1 (ld.global.cg).
#pragma once

#include "common.cuh"

namespace odi_cuda {

// Every kernel launched this way triggers its dependents on entry and waits for the
// kernels before it (griddepcontrol) before touching global memory, so all
// are launched with programmatic stream serialisation: the next kernel (a
// GEMV streaming its weights) may start while this one runs.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl_smem(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                                   Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, cudaStream_t s, Args... args) {
  return launch_pdl_smem(kern, grid, block, 0, s, args...);
}

}  // namespace odi_cuda
