// Cross attention: entry points, checks, launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstring>

#include "attention.h"

namespace mlxd {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxDims = MLXD_CROSS_MAX_HEAD_DIM / 32;   // of a head, for a lane

struct Heads {
  char* data;
  int64_t batch, token, head;   // strides in elements
};

struct CrossParams {
  Heads q, k, v, out, dout, dq, dk, dv;
  float* lse;
  float* delta;                 // [batch, q_heads, q_tokens]: sum of dout * out over a row
  const void* lengths;
  int lengths_dtype;
  const uint8_t* key_mask;
  int64_t key_mask_stride;
  int batch, q_tokens, kv_tokens, q_heads, kv_heads, group, head_dim;
  float scale;
};

__device__ int length_of(const CrossParams& p, int b) {
  if (!p.lengths) return p.kv_tokens;
  const int64_t n = p.lengths_dtype == MLXD_I64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
  return static_cast<int>(n < 0 ? 0 : n > p.kv_tokens ? p.kv_tokens : n);
}

__device__ bool is_read(const CrossParams& p, int b, int key) {
  return !p.key_mask || p.key_mask[b * p.key_mask_stride + key];
}

template <class T> __device__ const T* row_of(const Heads& h, int64_t b, int64_t s, int64_t head) {
  return reinterpret_cast<const T*>(h.data) + b * h.batch + s * h.token + head * h.head;
}

template <class T> __device__ T from_float(float v);
template <> __device__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T> __device__ void load_row(const T* x, int d, int lane, float (&v)[kMaxDims]) {
  for (int i = 0; i < kMaxDims; i++) v[i] = lane + 32 * i < d ? static_cast<float>(x[lane + 32 * i]) : 0.0f;
}

template <class T> __device__ void store_row(T* x, int d, int lane, const float (&v)[kMaxDims]) {
  for (int i = 0; i < kMaxDims; i++) {
    if (lane + 32 * i < d) x[lane + 32 * i] = from_float<T>(v[i]);
  }
}

__device__ float dot(const float (&a)[kMaxDims], const float (&b)[kMaxDims]) {
  float s = 0;
  for (int i = 0; i < kMaxDims; i++) s += a[i] * b[i];
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  return s;
}

// One warp a query row.
template <class T>
__global__ void __launch_bounds__(32 * kWarps) cross_forward_kernel(const __grid_constant__ CrossParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (id >= static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens) return;
  const int s = id % p.q_tokens, h = id / p.q_tokens % p.q_heads, b = id / p.q_tokens / p.q_heads;
  float q[kMaxDims], o[kMaxDims] = {}, m = -INFINITY, l = 0;
  load_row(row_of<T>(p.q, b, s, h), p.head_dim, lane, q);
  const int n = length_of(p, b);
  for (int key = 0; key < n; key++) {
    if (!is_read(p, b, key)) continue;
    float k[kMaxDims], v[kMaxDims];
    load_row(row_of<T>(p.k, b, key, h / p.group), p.head_dim, lane, k);
    load_row(row_of<T>(p.v, b, key, h / p.group), p.head_dim, lane, v);
    const float x = dot(q, k) * p.scale;
    const float top = fmaxf(m, x), keep = expf(m - top), e = expf(x - top);
    m = top;
    l = l * keep + e;
    for (int i = 0; i < kMaxDims; i++) o[i] = o[i] * keep + e * v[i];
  }
  for (int i = 0; i < kMaxDims; i++) o[i] = l > 0 ? o[i] / l : 0.0f;
  store_row(const_cast<T*>(row_of<T>(p.out, b, s, h)), p.head_dim, lane, o);
  if (p.lse && !lane) p.lse[id] = l > 0 ? m + logf(l) : -INFINITY;
}

// One warp a query row: its delta and the gradient of q.
template <class T>
__global__ void __launch_bounds__(32 * kWarps) cross_dq_kernel(const __grid_constant__ CrossParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (id >= static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens) return;
  const int s = id % p.q_tokens, h = id / p.q_tokens % p.q_heads, b = id / p.q_tokens / p.q_heads;
  float q[kMaxDims], o[kMaxDims], g[kMaxDims], dq[kMaxDims] = {};
  load_row(row_of<T>(p.q, b, s, h), p.head_dim, lane, q);
  load_row(row_of<T>(p.out, b, s, h), p.head_dim, lane, o);
  load_row(row_of<T>(p.dout, b, s, h), p.head_dim, lane, g);
  const float delta = dot(o, g), lse = p.lse[id];
  if (!lane) p.delta[id] = delta;
  const int n = length_of(p, b);
  for (int key = 0; key < n; key++) {
    if (!is_read(p, b, key)) continue;
    float k[kMaxDims], v[kMaxDims];
    load_row(row_of<T>(p.k, b, key, h / p.group), p.head_dim, lane, k);
    load_row(row_of<T>(p.v, b, key, h / p.group), p.head_dim, lane, v);
    const float w = expf(dot(q, k) * p.scale - lse), ds = w * (dot(g, v) - delta) * p.scale;
    for (int i = 0; i < kMaxDims; i++) dq[i] += ds * k[i];
  }
  store_row(const_cast<T*>(row_of<T>(p.dq, b, s, h)), p.head_dim, lane, dq);
}

// One warp a key: the gradients of k and v, summed over the query heads that share it.
template <class T>
__global__ void __launch_bounds__(32 * kWarps) cross_dkv_kernel(const __grid_constant__ CrossParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (id >= static_cast<int64_t>(p.batch) * p.kv_heads * p.kv_tokens) return;
  const int key = id % p.kv_tokens, hk = id / p.kv_tokens % p.kv_heads, b = id / p.kv_tokens / p.kv_heads;
  float k[kMaxDims], v[kMaxDims], dk[kMaxDims] = {}, dv[kMaxDims] = {};
  if (key < length_of(p, b) && is_read(p, b, key)) {
    load_row(row_of<T>(p.k, b, key, hk), p.head_dim, lane, k);
    load_row(row_of<T>(p.v, b, key, hk), p.head_dim, lane, v);
    for (int h = hk * p.group; h < (hk + 1) * p.group; h++) {
      for (int s = 0; s < p.q_tokens; s++) {
        const int64_t row = (static_cast<int64_t>(b) * p.q_heads + h) * p.q_tokens + s;
        float q[kMaxDims], g[kMaxDims];
        load_row(row_of<T>(p.q, b, s, h), p.head_dim, lane, q);
        load_row(row_of<T>(p.dout, b, s, h), p.head_dim, lane, g);
        const float w = expf(dot(q, k) * p.scale - p.lse[row]), ds = w * (dot(g, v) - p.delta[row]) * p.scale;
        for (int i = 0; i < kMaxDims; i++) {
          dv[i] += w * g[i];
          dk[i] += ds * q[i];
        }
      }
    }
  }
  store_row(const_cast<T*>(row_of<T>(p.dk, b, key, hk)), p.head_dim, lane, dk);
  store_row(const_cast<T*>(row_of<T>(p.dv, b, key, hk)), p.head_dim, lane, dv);
}

// Tensors as the copies into shared memory want them: 16-byte units throughout.  Strides of dimensions that are not
// stepped along do not matter.
bool aligned(const mlxd_heads& h, int batch, int tokens, int heads) {
  return reinterpret_cast<uintptr_t>(h.data) % 16 == 0 && (batch <= 1 || h.stride_batch % 8 == 0) &&
         (tokens <= 1 || h.stride_token % 8 == 0) && (heads <= 1 || h.stride_head % 8 == 0);
}

int check_sizes(const char* entry, const mlxd_cross_desc* d) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  if (!d) return bad("no descriptor");
  if (d->dtype != MLXD_BF16 && d->dtype != MLXD_F16) return bad("tensors must be bfloat16 or float16");
  if (d->batch < 0 || d->q_tokens < 0 || d->kv_tokens < 0) return bad("negative size");
  if (d->q_heads < 1 || d->kv_heads < 1 || d->q_heads % d->kv_heads) {
    return bad("q_heads must be a multiple of kv_heads (got " + std::to_string(d->q_heads) + " and " + std::to_string(d->kv_heads) + ")");
  }
  if (d->head_dim < 8 || d->head_dim % 8 || d->head_dim > MLXD_CROSS_MAX_HEAD_DIM) {
    return bad("head_dim must be a multiple of 8 up to " + std::to_string(MLXD_CROSS_MAX_HEAD_DIM) + " (got " + std::to_string(d->head_dim) + ")");
  }
  if (static_cast<int64_t>(d->batch) * d->q_heads > (1 << 24) || static_cast<int64_t>(d->batch) * d->q_heads * d->q_tokens > (int64_t{1} << 33)) {
    return bad("too many rows");
  }
  return MLXD_OK;
}

Heads heads_of(const mlxd_heads& h) {
  return Heads{static_cast<char*>(h.data), h.stride_batch, h.stride_token, h.stride_head};
}

int params_of(const char* entry, const mlxd_cross_desc* d, bool backward, CrossParams& p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  const int rc = check_sizes(entry, d);
  if (rc != MLXD_OK) return rc;
  if (!std::isfinite(d->scale)) return bad("scale must be finite");
  if (d->lengths && d->lengths_dtype != MLXD_I32 && d->lengths_dtype != MLXD_I64) return bad("lengths must be int32 or int64");
  const int b = d->batch, t = d->q_tokens, n = d->kv_tokens, hq = d->q_heads, hk = d->kv_heads;
  struct { const mlxd_heads* h; bool query; const char* name; } need[] = {
      {&d->q, true, "q"}, {&d->k, false, "k"}, {&d->v, false, "v"}, {&d->out, true, "out"},
      {&d->dout, true, "dout"}, {&d->dq, true, "dq"}, {&d->dk, false, "dk"}, {&d->dv, false, "dv"}};
  for (int i = 0; i < (backward ? 8 : 4); i++) {
    const auto& x = need[i];
    const int tokens = x.query ? t : n;
    if (!b || !tokens) continue;   // an empty tensor
    if (!x.h->data) return bad(std::string(x.name) + " is needed");
    if (!aligned(*x.h, b, tokens, x.query ? hq : hk)) {
      return bad(std::string(x.name) + " must start on 16 bytes and have strides that are multiples of 8");
    }
  }
  if (backward && b && t && !d->lse) return bad("lse is needed");
  std::memset(&p, 0, sizeof(p));
  p.q = heads_of(d->q);
  p.k = heads_of(d->k);
  p.v = heads_of(d->v);
  p.out = heads_of(d->out);
  p.dout = heads_of(d->dout);
  p.dq = heads_of(d->dq);
  p.dk = heads_of(d->dk);
  p.dv = heads_of(d->dv);
  p.lse = d->lse;
  p.lengths = d->lengths;
  p.lengths_dtype = d->lengths_dtype;
  p.key_mask = d->key_mask;
  p.key_mask_stride = d->key_mask_stride;
  p.batch = b;
  p.q_tokens = t;
  p.kv_tokens = n;
  p.q_heads = hq;
  p.kv_heads = hk;
  p.group = hq / hk;
  p.head_dim = d->head_dim;
  p.scale = d->scale;
  return MLXD_OK;
}

size_t workspace_bytes(const mlxd_cross_desc* d, bool backward) {
  return backward ? sizeof(float) * d->batch * d->q_heads * d->q_tokens : 0;
}

unsigned blocks_of(int64_t warps) {
  return static_cast<unsigned>((warps + kWarps - 1) / kWarps);
}

}  // namespace
}  // namespace mlxd

using namespace mlxd;

extern "C" int mlxd_cross_attention_workspace(int device, const mlxd_cross_desc* d, int backward, size_t* bytes) {
  return guarded("cross_attention_workspace", [&] {
    (void)device;
    const int rc = check_sizes("cross_attention_workspace", d);
    if (rc != MLXD_OK) return rc;
    if (!bytes) return fail(MLXD_ERR_INVALID, "cross_attention_workspace: no place for the result");
    *bytes = workspace_bytes(d, backward != 0);
    return static_cast<int>(MLXD_OK);
  });
}

extern "C" int mlxd_cross_attention(int device, void* cuda_stream, const mlxd_cross_desc* d) {
  return guarded("cross_attention", [&] {
    CrossParams p;
    const int rc = params_of("cross_attention", d, false, p);
    if (rc != MLXD_OK) return rc;
    const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens;
    if (!rows) return static_cast<int>(MLXD_OK);
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (d->dtype == MLXD_F16) cross_forward_kernel<__half><<<blocks_of(rows), 32 * kWarps, 0, s>>>(p);
    else cross_forward_kernel<__nv_bfloat16><<<blocks_of(rows), 32 * kWarps, 0, s>>>(p);
    MLXD_CUDA(cudaGetLastError());
    return static_cast<int>(MLXD_OK);
  });
}

extern "C" int mlxd_cross_attention_backward(int device, void* cuda_stream, const mlxd_cross_desc* d) {
  return guarded("cross_attention_backward", [&] {
    CrossParams p;
    const int rc = params_of("cross_attention_backward", d, true, p);
    if (rc != MLXD_OK) return rc;
    const size_t need = workspace_bytes(d, true);
    if (need && (!d->workspace || d->workspace_bytes < need)) return fail(MLXD_ERR_INVALID, "cross_attention_backward: workspace too small");
    p.delta = static_cast<float*>(d->workspace);
    const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens;
    const int64_t keys = static_cast<int64_t>(p.batch) * p.kv_heads * p.kv_tokens;
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (rows) {
      if (d->dtype == MLXD_F16) cross_dq_kernel<__half><<<blocks_of(rows), 32 * kWarps, 0, s>>>(p);
      else cross_dq_kernel<__nv_bfloat16><<<blocks_of(rows), 32 * kWarps, 0, s>>>(p);
      MLXD_CUDA(cudaGetLastError());
    }
    if (keys) {
      if (d->dtype == MLXD_F16) cross_dkv_kernel<__half><<<blocks_of(keys), 32 * kWarps, 0, s>>>(p);
      else cross_dkv_kernel<__nv_bfloat16><<<blocks_of(keys), 32 * kWarps, 0, s>>>(p);
      MLXD_CUDA(cudaGetLastError());
    }
    return static_cast<int>(MLXD_OK);
  });
}
