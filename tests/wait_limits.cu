// A wait that runs out: warps wait for a barrier that nothing arrives at, beside a warp whose products are awaited before tensor memory is
// freed.  Prints what the host checks; every wait here has its limit.
#include <cstdio>

#include "../mlx-data_b200/csrc/sm100.cuh"

using namespace mlxd;

struct Seen {
  int gave_up[4], failed, ended;
  unsigned long long ns;
};

__global__ void __launch_bounds__(128) wait_in_vain(Seen* seen) {
  __shared__ uint64_t bars[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t never = smem_address(bars), ended = never + 8;
  if (threadIdx.x == 0) {
    failed = 0;
    barrier_init(never, 1);
    barrier_init(ended, 1);
    barrier_init_done();
  }
  if (warp == 0) tmem_alloc<64>(smem_address(&tmem_slot));
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  unsigned long long from, to;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(from));
  const bool going = warp_wait(never, 0, &failed);
  if (warp == 0 && !going) products_end(ended);   // none are under way
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(to));
  if (lane == 0) seen->gave_up[warp] = !going;
  __syncthreads();
  if (warp == 0) tmem_free<64>(tmem_slot);
  if (threadIdx.x == 0) {
    seen->failed = failed;
    seen->ended = barrier_try(ended, 0);
    seen->ns = to - from;
  }
}

int main() {
  Seen* seen = nullptr;
  Seen got = {};
  cudaError_t e = cudaMalloc(&seen, sizeof(Seen));
  if (e == cudaSuccess) e = cudaMemset(seen, 0, sizeof(Seen));
  if (e == cudaSuccess) {
    wait_in_vain<<<1, 128>>>(seen);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(&got, seen, sizeof(Seen), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess) e = cudaFree(seen);
  printf("{\"status\": %d, \"gave_up\": [%d, %d, %d, %d], \"failed\": %d, \"ended\": %d, \"seconds\": %.3f}\n", e, got.gave_up[0],
         got.gave_up[1], got.gave_up[2], got.gave_up[3], got.failed, got.ended, got.ns * 1e-9);
  return e != cudaSuccess;
}
