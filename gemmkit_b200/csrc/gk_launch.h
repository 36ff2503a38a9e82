// gk_launch.h -- launching a plain kernel on a stream, overlapping the kernel before it where the
// engine's setting allows that (every kernel launched so waits with griddep_wait()).
#pragma once

#include <cuda_runtime.h>
#include <string.h>

#include "gk_engine.h"

namespace gk {

template <typename... P, typename... A>
int launch_overlapped_smem(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t st,
                           const A&... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = api_pdl_enabled() ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P(args)...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: kernel launch failed: %s", cudaGetErrorString(e));
    return GK_OK;
}

template <typename... P, typename... A>
int launch_overlapped(void (*kern)(P...), dim3 grid, int threads, cudaStream_t st, const A&... args) {
    return launch_overlapped_smem(kern, grid, threads, 0, st, args...);
}

}  // namespace gk
