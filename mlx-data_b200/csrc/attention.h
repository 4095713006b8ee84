// Host side shared by the attention operators: checks of descriptors and what their launches need.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <new>
#include <string>
#include <type_traits>

#include "../../include/mlxd_b200.h"
#include "context.h"

namespace mlxd {

struct Heads {
  char* data;
  int64_t batch, token, head;   // strides in elements
};

// bytes of an element; 0 for a type the operators do not take
inline int dtype_bytes(int dtype) {
  switch (dtype) {
    case MLXD_F32: case MLXD_I32: return 4;
    case MLXD_BF16: case MLXD_F16: return 2;
    case MLXD_I64: return 8;
    default: return 0;
  }
}

// Whether a pointer can be read in units of `bytes`; NULL can.
inline bool on_boundary(const void* p, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0;
}

// No exception leaves a C entry point.
template <class F>
int guarded(const char* entry, F&& body) {
  try {
    return body();
  } catch (const std::bad_alloc&) {
    return MLXD_ERR_NOMEM;
  } catch (const std::exception& e) {
    try {
      return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + e.what());
    } catch (...) {
      return MLXD_ERR_INVALID;
    }
  } catch (...) {
    return MLXD_ERR_INVALID;
  }
}

#ifdef __CUDACC__
// Launches a kernel that begins while the last CTAs of the kernel before it in the stream run, and that waits on the device
// (griddepcontrol.wait, in every CTA) for that one's end before it touches what others write or read.  Such a kernel reads by ordinary
// loads, not by those for memory that nobody writes while it runs.
template <class... Args>
cudaError_t launch_behind(void (*kernel)(Args...), dim3 grid, int threads, int bytes, cudaStream_t stream, int cluster, std::common_type_t<Args>... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute how[2] = {};
  how[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  how[0].val.programmaticStreamSerializationAllowed = 1;
  how[1].id = cudaLaunchAttributeClusterDimension;
  how[1].val.clusterDim.x = cluster;
  how[1].val.clusterDim.y = how[1].val.clusterDim.z = 1;
  config.attrs = how;
  config.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}
#endif

// SMs of a device, looked up once per device.
int device_sms(int device, int* sms);

}  // namespace mlxd
