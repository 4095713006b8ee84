// Cached and window attention, forward: a warp for each query and head, key by key, a running maximum and sum.
#include "causal.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;

template <class T, bool kPaged>
__global__ void __launch_bounds__(32 * kWarps) causal_forward_kernel(const __grid_constant__ CausalParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (row >= static_cast<int64_t>(p.batch) * p.q_heads * p.tokens) return;
  const int i = row % p.tokens, head = row / p.tokens % p.q_heads, b = row / p.tokens / p.q_heads, kv_head = head / p.group;
  const Sequence s = sequence_of<kPaged>(p, b);
  float q[4] = {}, o[4] = {}, top = -INFINITY, total = 0;
  const bool there = 4 * lane < p.head_dim;
  const auto load = [&](const char* data, int64_t at, float (&x)[4]) {
    const uint2 v = there ? *reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(data) + at + 4 * lane) : make_uint2(0, 0);
    const float2 lo = unpack2<T>(v.x), hi = unpack2<T>(v.y);
    x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
  };
  if (i < s.fresh) {
    load(p.q.data, b * p.q.batch + i * p.q.token + head * p.q.head, q);
    const float c = p.scale * kLog2e;
    const auto read = [&](int j) {
      int64_t major = b, minor = j;
      if (kPaged) {
        major = page_of(p.cache, b, j);
        minor = j & (p.cache.page_size - 1);
        if (major < 0) return;
      }
      float k[4], v[4];
      load(p.k.data, major * p.k.batch + minor * p.k.token + kv_head * p.k.head, k);
      load(p.v.data, major * p.v.batch + minor * p.v.token + kv_head * p.v.head, v);
      float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
      for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
      const float now = fmaxf(top, x);
      if (x == -INFINITY) return;
      const float keep = exp2_of((top - now) * c), w = exp2_of((x - now) * c);
      top = now;
      total = total * keep + w;
      for (int e = 0; e < 4; e++) o[e] = o[e] * keep + w * v[e];
    };
    int place = s.held + i, to = min(place + 1, s.end);
    const uint8_t* tree = p.tree ? p.tree + b * p.tree_batch + i * p.tree_token : nullptr;
    if (tree) {
      place = s.held;
      to = min(s.held, s.end);
      for (int j = 0; j < s.fresh; j++) place += j != i && tree[j];
    }
    const Reach r = reach_of(p, s, place, to);
    for (int j = 0; j < r.sinks; j++) read(j);
    for (int j = r.from; j < r.to; j++) read(j);
    if (tree) {
      for (int j = 0; j < s.fresh && s.held + j < s.end; j++) {
        if (tree[j]) read(s.held + j);
      }
    }
  }
  const float by = total == 0 ? 0.0f : 1.0f / total;
  if (there) {
    T* to = reinterpret_cast<T*>(p.out.data) + b * p.out.batch + i * p.out.token + head * p.out.head + 4 * lane;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(o[0] * by, o[1] * by), pack2<T>(o[2] * by, o[3] * by));
  }
  if (p.lse && lane == 0) p.lse[row] = total == 0 ? -INFINITY : top * p.scale + logf(total);
}

template <class T>
cudaError_t launch(const CausalParams& p, bool paged, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(p.batch) * p.q_heads * p.tokens + kWarps - 1) / kWarps);
  if (paged) causal_forward_kernel<T, true><<<blocks, 32 * kWarps, 0, stream>>>(p);
  else causal_forward_kernel<T, false><<<blocks, 32 * kWarps, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_causal_forward(const CausalParams& p, bool paged, int dtype, cudaStream_t stream) {
  return dtype == MLXD_F16 ? launch<__half>(p, paged, stream) : launch<__nv_bfloat16>(p, paged, stream);
}

}  // namespace mlxd
