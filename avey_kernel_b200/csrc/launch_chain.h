// The launches of one call, in order on one stream: all but the first may be set up
// beside the end of the one before. Every kernel launched so, those that are the first of
// all their calls too, waits for that one (griddepcontrol.wait) ahead of its first read, in every
// thread, so what an earlier launch wrote is seen by all later ones.
#pragma once

#include <cuda_runtime.h>

#include <cstdio>

#include "avey_b200.h"
#include "host_api.h"

namespace avey_host {

struct Chain {
  cudaStream_t stream;
  bool after = false;

  template <typename... Params, typename... Args>
  int launch(const char* what, void (*kernel)(Params...), dim3 grid, int block, int smem, int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
      attr[n].id = cudaLaunchAttributeClusterDimension;
      attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
      attr[n].val.clusterDim.y = 1;
      attr[n].val.clusterDim.z = 1;
      ++n;
    }
    if (after) {
      attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[n].val.programmaticStreamSerializationAllowed = 1;
      ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(n);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
    if (e != cudaSuccess) {
      char buf[256];
      snprintf(buf, sizeof(buf), "%s launch: %s", what, cudaGetErrorString(e));
      return set_error(AVEY_ERR_LAUNCH, buf);
    }
    count_launches(1);
    after = true;
    return AVEY_OK;
  }
};

}  // namespace avey_host
