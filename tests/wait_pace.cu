// Waits for something far off.  In CTA 0 a warp counts its progress for four seconds and then arrives; in CTA 1 it stops counting after one and
// never does.  One warp waits behind the count, another as if it were next.  Prints what the host checks; every wait here has its limit.
#include <cstdio>

#include "../mlx-data_b200/csrc/sm100.cuh"

using namespace mlxd;

struct Seen {
  int came[2];
  float seconds[2];
};

__device__ unsigned long long now() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

__global__ void __launch_bounds__(96) waits(Seen* seen) {
  __shared__ uint64_t bar;
  __shared__ uint32_t progress;
  __shared__ int failed[2];
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    progress = failed[0] = failed[1] = 0;
    barrier_init(smem_address(&bar), 1);
    barrier_init_done();
  }
  __syncthreads();
  const unsigned long long from = now();
  if (warp == 2) {
    if (lane == 0) {
      const int steps = blockIdx.x ? 4 : 16;   // a quarter of a second each, and no more than so many naps
      for (int i = 1; i <= steps; i++) {
        for (int nap = 0; nap < 1000000 && now() - from < i * 250000000ull; nap++) __nanosleep(10000);
        *static_cast<volatile uint32_t*>(&progress) = i;
      }
      if (blockIdx.x == 0) barrier_arrive(smem_address(&bar));
    }
  } else {
    const bool came = warp ? warp_wait(smem_address(&bar), 0, &failed[1]) : warp_wait_behind(smem_address(&bar), 0, &failed[0], &progress);
    if (lane == 0) {
      seen[blockIdx.x].came[warp] = came && !failed[warp];
      seen[blockIdx.x].seconds[warp] = (now() - from) * 1e-9f;
    }
  }
}

int main() {
  Seen* seen = nullptr;
  Seen got[2] = {};
  cudaError_t e = cudaMalloc(&seen, sizeof(got));
  if (e == cudaSuccess) {
    waits<<<2, 96>>>(seen);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(got, seen, sizeof(got), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess) e = cudaFree(seen);
  printf("{\"status\": %d, \"came\": [%d, %d, %d, %d], \"seconds\": [%.3f, %.3f, %.3f, %.3f]}\n", e, got[0].came[0], got[0].came[1],
         got[1].came[0], got[1].came[1], got[0].seconds[0], got[0].seconds[1], got[1].seconds[0], got[1].seconds[1]);
  return e != cudaSuccess;
}
