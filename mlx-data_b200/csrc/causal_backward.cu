// Gradients of window attention: a warp for each query and head, then a warp for each key and head.
#include "causal.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;

template <class T>
__device__ __forceinline__ void load4(const Heads& x, int b, int i, int head, int lane, bool there, float (&to)[4]) {
  const T* at = reinterpret_cast<const T*>(x.data) + b * x.batch + i * x.token + head * x.head + 4 * lane;
  const uint2 v = there ? *reinterpret_cast<const uint2*>(at) : make_uint2(0, 0);
  const float2 lo = unpack2<T>(v.x), hi = unpack2<T>(v.y);
  to[0] = lo.x, to[1] = lo.y, to[2] = hi.x, to[3] = hi.y;
}

template <class T>
__device__ __forceinline__ void store4(const Heads& x, int b, int i, int head, int lane, bool there, const float (&v)[4], float by) {
  T* at = reinterpret_cast<T*>(x.data) + b * x.batch + i * x.token + head * x.head + 4 * lane;
  if (there) *reinterpret_cast<uint2*>(at) = make_uint2(pack2<T>(v[0] * by, v[1] * by), pack2<T>(v[2] * by, v[3] * by));
}

__device__ __forceinline__ float dot4(const float (&a)[4], const float (&b)[4]) {
  float x = a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
  return x;
}

// dQ = scale dS K, dS = P (dP - delta), delta = sum(dO O) - dlse, which the other kernel reads.
template <class T>
__global__ void __launch_bounds__(32 * kWarps) causal_dq_kernel(const __grid_constant__ CausalParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (row >= static_cast<int64_t>(p.batch) * p.q_heads * p.tokens) return;
  const int i = row % p.tokens, head = row / p.tokens % p.q_heads, b = row / p.tokens / p.q_heads, kv_head = head / p.group;
  const bool there = 4 * lane < p.head_dim;
  const Sequence s = sequence_of<false>(p, b);
  float dq[4] = {};
  if (i < s.fresh) {
    float q[4], o[4], g[4];
    load4<T>(p.q, b, i, head, lane, there, q);
    load4<T>(p.out, b, i, head, lane, there, o);
    load4<T>(p.dout, b, i, head, lane, there, g);
    const float delta = dot4(o, g) - (p.lse_grad ? p.lse_grad[row] : 0.0f), base = row_base(p.lse[row]);
    if (lane == 0) p.delta[row] = delta;
    const Reach r = reach_of(p, s, i, i + 1);
    for (int j = r.sinks ? 0 : r.from; j < r.to; j = j + 1 == r.sinks ? r.from : j + 1) {
      float k[4], v[4];
      load4<T>(p.k, b, j, kv_head, lane, there, k);
      load4<T>(p.v, b, j, kv_head, lane, there, v);
      const float ds = exp2_of(dot4(q, k) * p.scale * kLog2e + base) * (dot4(g, v) - delta);
      for (int e = 0; e < 4; e++) dq[e] += ds * k[e];
    }
  }
  store4<T>(p.dq, b, i, head, lane, there, dq, p.scale);
}

// dV = P^T dO, dK = scale dS^T Q, over the queries of every head that shares the key.
template <class T>
__global__ void __launch_bounds__(32 * kWarps) causal_dkv_kernel(const __grid_constant__ CausalParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (row >= static_cast<int64_t>(p.batch) * p.kv_heads * p.tokens) return;
  const int j = row % p.tokens, kv_head = row / p.tokens % p.kv_heads, b = row / p.tokens / p.kv_heads;
  const bool there = 4 * lane < p.head_dim;
  const Sequence s = sequence_of<false>(p, b);
  float dk[4] = {}, dv[4] = {};
  if (j < s.fresh) {
    float k[4], v[4];
    load4<T>(p.k, b, j, kv_head, lane, there, k);
    load4<T>(p.v, b, j, kv_head, lane, there, v);
    const int end = j < p.sinks || p.window > s.fresh - j ? s.fresh : j + p.window;
    for (int head = kv_head * p.group; head < (kv_head + 1) * p.group; head++) {
      for (int i = j; i < end; i++) {
        const int64_t stat = (static_cast<int64_t>(b) * p.q_heads + head) * p.tokens + i;
        float q[4], g[4];
        load4<T>(p.q, b, i, head, lane, there, q);
        load4<T>(p.dout, b, i, head, lane, there, g);
        const float w = exp2_of(dot4(q, k) * p.scale * kLog2e + row_base(p.lse[stat])), ds = w * (dot4(g, v) - p.delta[stat]);
        for (int e = 0; e < 4; e++) {
          dv[e] += w * g[e];
          dk[e] += ds * q[e];
        }
      }
    }
  }
  store4<T>(p.dk, b, j, kv_head, lane, there, dk, p.scale);
  store4<T>(p.dv, b, j, kv_head, lane, there, dv, 1.0f);
}

template <class T>
cudaError_t launch(const CausalParams& p, cudaStream_t stream) {
  const auto blocks = [&](int heads) { return static_cast<unsigned>((static_cast<int64_t>(p.batch) * heads * p.tokens + kWarps - 1) / kWarps); };
  causal_dq_kernel<T><<<blocks(p.q_heads), 32 * kWarps, 0, stream>>>(p);
  causal_dkv_kernel<T><<<blocks(p.kv_heads), 32 * kWarps, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_causal_backward(const CausalParams& p, int dtype, cudaStream_t stream) {
  return dtype == MLXD_F16 ? launch<__half>(p, stream) : launch<__nv_bfloat16>(p, stream);
}

}  // namespace mlxd
