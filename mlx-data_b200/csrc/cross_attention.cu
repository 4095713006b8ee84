// Cross attention: entry points, checks, launches.
#include <cmath>
#include <cstring>

#include "attention.h"
#include "cross.h"

namespace mlxd {

namespace {

// Set by a kernel whose wait for its own copies or products ran out, and never cleared: whoever asks learns of it, on any stream.
__device__ int attention_status;

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
  if (d->q_tokens > (1 << 30) || d->kv_tokens > (1 << 30)) return bad("more than 2^30 tokens");
  if (static_cast<int64_t>(d->batch) * d->q_heads > (1 << 24) || static_cast<int64_t>(d->batch) * d->q_heads * d->q_tokens > (int64_t{1} << 33)) {
    return bad("too many rows");
  }
  if (static_cast<int64_t>(d->batch) * d->kv_heads * ((static_cast<int64_t>(d->kv_tokens) + 127) / 128) > INT32_MAX) return bad("too many keys");
  return MLXD_OK;
}

Heads heads_of(const mlxd_heads& h) {
  return Heads{static_cast<char*>(h.data), h.stride_batch, h.stride_token, h.stride_head};
}

CrossParams sizes_of(const mlxd_cross_desc* d) {
  CrossParams p;
  std::memset(&p, 0, sizeof(p));
  p.batch = d->batch;
  p.q_tokens = d->q_tokens;
  p.kv_tokens = d->kv_tokens;
  p.q_heads = d->q_heads;
  p.kv_heads = d->kv_heads;
  p.group = d->q_heads / d->kv_heads;
  p.head_dim = d->head_dim;
  p.scale = d->scale;
  return p;
}

int workspace_of(int device, const CrossParams& p, bool backward, size_t* bytes) {
  *bytes = 0;
  if (backward) {
    *bytes = sizeof(float) * p.batch * p.q_heads * p.q_tokens;
  } else if (p.batch && p.q_tokens) {
    int sms = 0;
    const int rc = device_sms(device, &sms);
    if (rc != MLXD_OK) return rc;
    if (takes_steps(p, sms)) *bytes = step_workspace(p, sms);
  }
  return MLXD_OK;
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
  // a kernel reads and writes whole elements, and a misaligned one is a fault
  if (!on_boundary(d->lse, 4)) return bad("lse does not start on a multiple of 4 bytes");
  if (d->lengths && !on_boundary(d->lengths, dtype_bytes(d->lengths_dtype))) return bad("lengths do not start on a multiple of their element's size");
  if (!on_boundary(d->workspace, 16)) return bad("workspace must start on 16 bytes");
  p = sizes_of(d);
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
  return MLXD_OK;
}

// Maps of the tensors that a pass copies or stores by tiles; those of empty tensors are left as they are.
int maps_of(const CrossParams& p, int dtype, bool backward, CrossMaps& m) {
  struct { const Heads* h; bool query; CUtensorMap* map; } all[] = {
      {&p.q, true, &m.q}, {&p.k, false, &m.k}, {&p.v, false, &m.v}, {&p.out, true, &m.out},
      {&p.dout, true, &m.dout}, {&p.dq, true, &m.dq}, {&p.dk, false, &m.dk}, {&p.dv, false, &m.dv}};
  for (int i = 0; i < (backward ? 8 : 4); i++) {
    const auto& x = all[i];
    const int tokens = x.query ? p.q_tokens : p.kv_tokens;
    if (!tokens || (backward && i == 3)) continue;
    const int rc = cross_map(*x.h, dtype, p.device, p.batch, tokens, x.query ? p.q_heads : p.kv_heads, p.head_dim, x.map);
    if (rc != MLXD_OK) return rc;
  }
  return MLXD_OK;
}

}  // namespace

int status_word(int device, int** word) {
  constexpr int kDevices = 64;
  static std::atomic<int*> known[kDevices];
  if (device < 0 || device >= kDevices) return fail(MLXD_ERR_INVALID, "device index out of range");
  *word = known[device].load(std::memory_order_relaxed);
  if (!*word) {
    void* at = nullptr;
    MLXD_CUDA(cudaGetSymbolAddress(&at, static_cast<const void*>(&attention_status)));
    *word = static_cast<int*>(at);
    known[device].store(*word, std::memory_order_relaxed);
  }
  return MLXD_OK;
}

// The driver's encoder, found through the runtime: the library links against no driver library.
int tile_map(const char* entry, int dtype, int device, void* data, int rank, const uint64_t* sizes, const int64_t* strides, const uint32_t* box,
             CUtensorMap* map) {
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
  cuuint64_t dims[5], bytes[4];
  cuuint32_t boxes[5];
  const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; i++) {
    dims[i] = sizes[i];
    boxes[i] = box[i];
    // strides of dimensions that are not stepped along may be anything; the encoder wants multiples of 16 bytes
    if (i) bytes[i - 1] = static_cast<cuuint64_t>(sizes[i] > 1 ? strides[i] * 2 : 16);
  }
  const auto make = [&] {
    return encode(map, dtype == MLXD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank), data,
                  dims, bytes, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = make();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
    // a thread that has not used CUDA before: the runtime binds the device's context to it, the driver's encoder does not
    MLXD_CUDA(cudaSetDevice(device));
    r = make();
  }
  if (r == CUDA_ERROR_INVALID_VALUE) return fail(MLXD_ERR_INVALID, std::string(entry) + ": a tensor's strides do not fit a tensor map");
  if (r != CUDA_SUCCESS) return fail(MLXD_ERR_CUDA, std::string(entry) + ": no tensor map (driver status " + std::to_string(r) + ")");
  return MLXD_OK;
}

int cross_map(const Heads& h, int dtype, int device, int batch, int tokens, int heads, int dim, CUtensorMap* map) {
  const uint64_t sizes[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(tokens), static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const int64_t strides[4] = {1, h.token, h.head, h.batch};
  const uint32_t box[4] = {64, 128, 1, 1};
  return tile_map("cross_attention", dtype, device, h.data, 4, sizes, strides, box, map);
}

}  // namespace mlxd

using namespace mlxd;

extern "C" int mlxd_cross_attention_workspace(int device, const mlxd_cross_desc* d, int backward, size_t* bytes) {
  return guarded("cross_attention_workspace", [&] {
    int rc = check_sizes("cross_attention_workspace", d);
    if (rc != MLXD_OK) return rc;
    if (!bytes) return fail(MLXD_ERR_INVALID, "cross_attention_workspace: no place for the result");
    return workspace_of(device, sizes_of(d), backward != 0, bytes);
  });
}

extern "C" int mlxd_cross_attention(int device, void* cuda_stream, const mlxd_cross_desc* d) {
  return guarded("cross_attention", [&] {
    CrossParams p;
    int rc = params_of("cross_attention", d, false, p);
    if (rc != MLXD_OK) return rc;
    if (!p.batch || !p.q_tokens) return static_cast<int>(MLXD_OK);
    size_t need = 0;
    rc = workspace_of(device, p, false, &need);
    if (rc != MLXD_OK) return rc;
    if (need && (!d->workspace || d->workspace_bytes < need)) return fail(MLXD_ERR_INVALID, "cross_attention: workspace too small");
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    p.device = device;
    int sms = 0;
    rc = device_sms(device, &sms);
    if (rc != MLXD_OK) return rc;
    if (takes_steps(p, sms)) {
      MLXD_CUDA(launch_cross_step(p, d->workspace, sms, d->dtype, s));
      return static_cast<int>(MLXD_OK);
    }
    rc = status_word(device, &p.status);
    CrossMaps maps;
    if (rc == MLXD_OK) rc = maps_of(p, d->dtype, false, maps);
    if (rc != MLXD_OK) return rc;
    MLXD_CUDA(launch_cross_forward(p, maps, d->dtype, s));
    return static_cast<int>(MLXD_OK);
  });
}

extern "C" int mlxd_cross_attention_backward(int device, void* cuda_stream, const mlxd_cross_desc* d) {
  return mlxd_cross_attention_backward_lse(device, cuda_stream, d, nullptr);
}

extern "C" int mlxd_cross_attention_backward_lse(int device, void* cuda_stream, const mlxd_cross_desc* d, const float* lse_grad) {
  return guarded("cross_attention_backward", [&] {
    CrossParams p;
    int rc = params_of("cross_attention_backward", d, true, p);
    if (rc != MLXD_OK) return rc;
    if (!on_boundary(lse_grad, 4)) return fail(MLXD_ERR_INVALID, "cross_attention_backward: lse_grad does not start on a multiple of 4 bytes");
    p.lse_grad = lse_grad;
    size_t need = 0;
    rc = workspace_of(device, p, true, &need);
    if (rc != MLXD_OK) return rc;
    if (need && (!d->workspace || d->workspace_bytes < need)) return fail(MLXD_ERR_INVALID, "cross_attention_backward: workspace too small");
    p.delta = static_cast<float*>(d->workspace);
    if (!p.batch) return static_cast<int>(MLXD_OK);
    MLXD_ON_DEVICE(device);
    p.device = device;
    rc = status_word(device, &p.status);
    CrossMaps maps;
    if (rc == MLXD_OK) rc = maps_of(p, d->dtype, true, maps);
    if (rc != MLXD_OK) return rc;
    MLXD_CUDA(launch_cross_backward(p, maps, d->dtype, static_cast<cudaStream_t>(cuda_stream)));
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
    MLXD_CUDA(cudaStreamSynchronize(s));
    *status = got;
    return got ? fail(MLXD_ERR_DEVICE, "attention: a kernel gave up waiting for its own copies or products; its results are not valid") : static_cast<int>(MLXD_OK);
  });
}
