// What the parts of cross attention share.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/mlxd_b200.h"

namespace mlxd {

struct Heads {
  char* data;
  int64_t batch, token, head;   // strides in elements
};

struct CrossParams {
  Heads q, k, v, out, dout, dq, dk, dv;
  float* lse;
  const float* lse_grad;        // backward: the gradient of lse, or null
  float* delta;                 // [batch, q_heads, q_tokens]: sum of dout * out over a row, less the gradient of its lse
  const void* lengths;
  int lengths_dtype;
  const uint8_t* key_mask;
  int64_t key_mask_stride;
  int batch, q_tokens, kv_tokens, q_heads, kv_heads, group, head_dim;
  float scale;
  int* status;                  // set where a wait ran out
  int device;
};

// Tensor maps of a call: boxes of 64 elements by 128 tokens, 128-byte swizzle.
struct CrossMaps {
  CUtensorMap q, k, v, out, dout, dq, dk, dv;   // forward: the first four; backward: all but out
};

// Raises a kernel's limit of shared memory, once per device.
template <auto kKernel>
cudaError_t allow_shared(int bytes, int device) {
  static std::atomic<uint64_t> done{0};   // of this kernel, a bit for each device
  const uint64_t bit = uint64_t{1} << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

int cross_map(const Heads& h, int dtype, int device, int batch, int tokens, int heads, int dim, CUtensorMap* map);

cudaError_t launch_cross_forward(const CrossParams& p, const CrossMaps& maps, int dtype, cudaStream_t stream);

// Few queries: whether a call is one, and how it runs.
bool takes_steps(const CrossParams& p, int sms);
size_t step_workspace(const CrossParams& p, int sms);
cudaError_t launch_cross_step(const CrossParams& p, void* workspace, int sms, int dtype, cudaStream_t stream);

cudaError_t launch_cross_backward(const CrossParams& p, const CrossMaps& maps, int dtype, cudaStream_t stream);

#ifdef __CUDACC__
// What a row's scores c s are added to in the backward pass, so that 2^(c s + base) is its weight.  A row whose scores are all -infinity
// has no weights: 0, as in the forward pass, not the infinity less infinity that its lse would give.
__device__ __forceinline__ float row_base(float lse) { return lse == -INFINITY ? -INFINITY : -lse * 1.4426950408889634f; }

__device__ __forceinline__ int length_of(const CrossParams& p, int b) {
  if (!p.lengths) return p.kv_tokens;
  const int64_t n = p.lengths_dtype == MLXD_I64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
  return static_cast<int>(n < 0 ? 0 : n > p.kv_tokens ? p.kv_tokens : n);
}

// The number of the CTA, read anew: what follows from it at a kernel's end is worked out again there instead of held in registers (forward,
// 6 x 333 tokens, 1024 keys, 16 heads of 64: 34.5 us with it held and spills, 32.9 without).
__device__ __forceinline__ int block_again() {
  int x;
  asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(x));
  return x;
}

// What a CTA that gave up leaves in rows `first` to `end` - 1 of a head, with all its threads: not a number (of either 16-bit type), instead
// of whatever the memory held.
__device__ __forceinline__ void spoil_rows(const Heads& x, int batch, int head, int first, int end, int dim) {
  for (int row = first + static_cast<int>(threadIdx.x) / 32; row < end; row += static_cast<int>(blockDim.x) / 32) {
    uint16_t* to = reinterpret_cast<uint16_t*>(x.data) + batch * x.batch + row * x.token + head * x.head;
    for (int i = threadIdx.x & 31; i < dim; i += 32) to[i] = 0x7fff;
  }
}

// The end of a sample's last key that is read, found by the whole CTA from the back: the padding below the images of a batch
// ends a sample's keys under a mask too.  `reach` (shared) is 0 before, for all threads.
__device__ __forceinline__ int reach_of(const CrossParams& p, int b, int length, int* reach) {
  if (!p.key_mask) return length;
  const uint8_t* mask = p.key_mask + b * p.key_mask_stride;
  for (int end = length; end > 0; end -= blockDim.x) {
    const int key = end - 1 - static_cast<int>(threadIdx.x);
    const int most = __reduce_max_sync(~0u, key >= 0 && mask[key] ? key + 1 : 0);
    if (most && (threadIdx.x & 31) == 0) atomicMax(reach, most);
    __syncthreads();
    const int found = *reach;
    __syncthreads();
    if (found) return found;
  }
  return 0;
}
#endif

}  // namespace mlxd
