// Host side shared by the grouped-query operators' entry points.
#pragma once

#include <algorithm>
#include <cstdio>

#include "../../../../include/dsv41_b200.h"
#include "common.cuh"

namespace dsv41 {

template <class T>
T* ptr(int64_t v) {
  return reinterpret_cast<T*>(v);
}

inline int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One launch with programmatic dependent launch (every kernel waits before it reads).
template <class... Exp, class... Args>
int launch(void (*kernel)(Exp...), dim3 grid, dim3 block, int smem, void* stream, const Args&... args) {
  cudaError_t e = smem > 48 * 1024 ? ensure_smem(reinterpret_cast<const void*>(kernel), smem) : cudaSuccess;
  if (e == cudaSuccess) {
    count_launch();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_on() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, args...);
  }
  if (e == cudaSuccess) return DSV41_OK;
  cudaGetLastError();
  fprintf(stderr, "dsv41: launch failed: %s\n", cudaGetErrorString(e));
  return DSV41_ELAUNCH;
}

}  // namespace dsv41
