// A wait that runs out: warps wait for a barrier that nothing arrives at, beside a warp whose products are awaited before tensor memory is
// freed, and leave rows of a tensor that are not numbers.  Prints what the host checks; every wait here has its limit.
#include <cstdio>

#include <vector>

#include "../mlx-data_b200/csrc/cross.h"
#include "../mlx-data_b200/csrc/sm100.cuh"

using namespace mlxd;

struct Seen {
  int gave_up[4], failed, ended;
  unsigned long long ns;
};

// [2 samples, 300 tokens, 3 heads, 24 of 40 elements]; the kernel gives up rows 128 to 255 of head 1 of sample 1
constexpr int kTokens = 300, kHeads = 3, kDim = 24, kRow = 40, kSize = 2 * kTokens * kHeads * kRow;

__global__ void __launch_bounds__(128) wait_in_vain(Seen* seen, Heads x) {
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
  if (failed) spoil_rows(x, 1, 1, 128, 256, kDim);
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
  uint16_t* x = nullptr;
  if (e == cudaSuccess) e = cudaMalloc(&x, sizeof(uint16_t) * kSize);
  if (e == cudaSuccess) e = cudaMemset(x, 0, sizeof(uint16_t) * kSize);
  if (e == cudaSuccess) {
    wait_in_vain<<<1, 128>>>(seen, Heads{reinterpret_cast<char*>(x), kTokens * kHeads * kRow, kHeads * kRow, kRow});
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(&got, seen, sizeof(Seen), cudaMemcpyDeviceToHost);
  std::vector<uint16_t> rows(kSize);
  if (e == cudaSuccess) e = cudaMemcpy(rows.data(), x, sizeof(uint16_t) * kSize, cudaMemcpyDeviceToHost);
  int spoiled = 0, wrong = 0;
  for (int i = 0; i < kSize; i++) {
    const int element = i % kRow, head = i / kRow % kHeads, token = i / kRow / kHeads % kTokens, batch = i / kRow / kHeads / kTokens;
    const bool mine = batch == 1 && head == 1 && token >= 128 && token < 256 && element < kDim;
    spoiled += mine && rows[i] == 0x7fff;
    wrong += !mine && rows[i] != 0;
  }
  if (e == cudaSuccess) e = cudaFree(x);
  if (e == cudaSuccess) e = cudaFree(seen);
  printf("{\"status\": %d, \"gave_up\": [%d, %d, %d, %d], \"failed\": %d, \"ended\": %d, \"seconds\": %.3f, \"spoiled\": %d, \"wrong\": %d}\n", e, got.gave_up[0],
         got.gave_up[1], got.gave_up[2], got.gave_up[3], got.failed, got.ended, got.ns * 1e-9,
         spoiled, wrong);
  return e != cudaSuccess;
}
