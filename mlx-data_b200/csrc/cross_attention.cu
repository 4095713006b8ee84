// Cross attention: entry points, checks, launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstring>

#include "attention.h"
#include "cross.h"

namespace mlxd {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxDims = MLXD_CROSS_MAX_HEAD_DIM / 32;   // of a head, for a lane

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

// Set by a kernel whose wait for its own copies or products ran out.
__device__ int attention_status;

int status_word(int device, int** word) {
  constexpr int kDevices = 64;
  static std::atomic<int*> known[kDevices];
  if (device < 0 || device >= kDevices) return fail(MLXD_ERR_INVALID, "device index out of range");
  *word = known[device].load(std::memory_order_relaxed);
  if (!*word) {
    void* at = nullptr;
    MLXD_CUDA(cudaGetSymbolAddress(&at, attention_status));
    *word = static_cast<int*>(at);
    known[device].store(*word, std::memory_order_relaxed);
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
  if (!std::isfinite(d->scale) || d->scale <= 0) return bad("scale must be positive and finite");
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

// The driver's encoder, found through the runtime: the library links against no driver library.
int cross_map(const Heads& h, int dtype, int batch, int tokens, int heads, int dim, CUtensorMap* map) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};
  Encode encode = known.load(std::memory_order_relaxed);
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    MLXD_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !f) return fail(MLXD_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    encode = reinterpret_cast<Encode>(f);
    known.store(encode, std::memory_order_relaxed);
  }
  const cuuint64_t sizes[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(batch)};
  // strides of dimensions that are not stepped along may be anything; the encoder wants multiples of 16 bytes
  const auto bytes = [](int64_t stride, int size) { return static_cast<cuuint64_t>(size > 1 ? stride * 2 : 16); };
  const cuuint64_t strides[3] = {bytes(h.token, tokens), bytes(h.head, heads), bytes(h.batch, batch)};
  const cuuint32_t box[4] = {64, 128, 1, 1}, steps[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, dtype == MLXD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, h.data, sizes,
                            strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MLXD_ERR_INVALID, "cross_attention: a tensor's strides do not fit a tensor map (status " + std::to_string(r) + ")");
  return MLXD_OK;
}

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
    int rc = params_of("cross_attention", d, false, p);
    if (rc != MLXD_OK) return rc;
    if (!p.batch || !p.q_tokens) return static_cast<int>(MLXD_OK);
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    rc = status_word(device, &p.status);
    CrossMaps maps;
    if (rc == MLXD_OK) rc = cross_map(p.q, d->dtype, p.batch, p.q_tokens, p.q_heads, p.head_dim, &maps.q);
    if (rc == MLXD_OK) rc = cross_map(p.out, d->dtype, p.batch, p.q_tokens, p.q_heads, p.head_dim, &maps.out);
    if (rc == MLXD_OK && p.kv_tokens) rc = cross_map(p.k, d->dtype, p.batch, p.kv_tokens, p.kv_heads, p.head_dim, &maps.k);
    if (rc == MLXD_OK && p.kv_tokens) rc = cross_map(p.v, d->dtype, p.batch, p.kv_tokens, p.kv_heads, p.head_dim, &maps.v);
    if (rc != MLXD_OK) return rc;
    MLXD_CUDA(launch_cross_forward(p, maps, d->dtype, s));
    return static_cast<int>(MLXD_OK);
  });
}

extern "C" int mlxd_attention_status(int device, void* cuda_stream, int32_t* status) {
  return guarded("attention_status", [&] {
    if (!status) return fail(MLXD_ERR_INVALID, "attention_status: no place for the result");
    MLXD_ON_DEVICE(device);
    int* word = nullptr;
    const int rc = status_word(device, &word);
    if (rc != MLXD_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    int32_t got = 0;
    MLXD_CUDA(cudaMemcpyAsync(&got, word, sizeof(got), cudaMemcpyDeviceToHost, s));
    MLXD_CUDA(cudaMemsetAsync(word, 0, sizeof(got), s));
    MLXD_CUDA(cudaStreamSynchronize(s));
    *status = got;
    return got ? fail(MLXD_ERR_DEVICE, "attention: a kernel gave up waiting for its own copies or products; its results are not valid") : static_cast<int>(MLXD_OK);
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
