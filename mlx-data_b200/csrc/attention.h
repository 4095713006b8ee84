// Host side shared by the attention operators: checks of descriptors and what their launches need.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <new>
#include <string>

#include "../../include/mlxd_b200.h"
#include "context.h"

namespace mlxd {

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

// SMs of a device, looked up once per device.
int device_sms(int device, int* sms);

}  // namespace mlxd
