// Rotary positions with several axes, alone or behind a norm of every head, forward and backward.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>

#include "attention.h"

namespace mlxd {

namespace {

constexpr int kWarps = 4;                                // of a CTA
constexpr int kMaxPairs = MLXD_ROTARY_MAX_HEAD_DIM / 2;

struct Heads {
  char* data;
  int64_t batch, token, head;   // strides in elements
};

struct RotaryParams {
  Heads q, k, q_out, k_out, q_grad, k_grad;
  const void* positions;
  int64_t pos_axis, pos_batch, pos_token;
  const float* frequencies;
  const void* q_weight;
  const void* k_weight;
  float* partial;               // [blocks][2][head_dim] sums of the weights' gradients
  int64_t rows;                 // batch * tokens
  int tokens, q_heads, k_heads, head_dim, pairs;
  int positions_dtype, weight_dtype, adjacent;
  float sign, eps;              // sign: -1 turns back
  uint32_t axes[kMaxPairs / 16];   // axis of a pair, two bits each
};

template <class T> __device__ float to_float(T v) { return static_cast<float>(v); }
template <class T> __device__ T from_float(float v);
template <> __device__ float from_float<float>(float v) { return v; }
template <> __device__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ float weight_at(const void* w, int dtype, int i) {
  if (!w) return 1.0f;
  if (dtype == MLXD_F32) return static_cast<const float*>(w)[i];
  if (dtype == MLXD_F16) return to_float(static_cast<const __half*>(w)[i]);
  return to_float(static_cast<const __nv_bfloat16*>(w)[i]);
}

__device__ float position_at(const RotaryParams& p, int axis, int64_t b, int64_t s) {
  const int64_t at = axis * p.pos_axis + b * p.pos_batch + s * p.pos_token;
  if (p.positions_dtype == MLXD_I64) return static_cast<float>(static_cast<const int64_t*>(p.positions)[at]);
  if (p.positions_dtype == MLXD_I32) return static_cast<float>(static_cast<const int32_t*>(p.positions)[at]);
  return static_cast<const float*>(p.positions)[at];
}

// The angle is the float32 product by definition; sincosf reduces arguments of any size.
__device__ float2 unit_of(const RotaryParams& p, int pair, int64_t b, int64_t s) {
  if (pair >= p.pairs) return make_float2(1.0f, 0.0f);
  const int axis = p.axes[pair >> 4] >> (2 * (pair & 15)) & 3;
  float2 u;
  sincosf(__fmul_rn(position_at(p, axis, b, s), p.frequencies[pair]), &u.y, &u.x);
  u.y *= p.sign;
  return u;
}

// Elements of pair i of a head; pairs beyond p.pairs are the elements that pass through, two by two.
__device__ void elements_of(const RotaryParams& p, int i, int& lo, int& hi) {
  if (p.adjacent) {
    lo = 2 * i;
    hi = 2 * i + 1;
  } else if (i < p.pairs) {
    lo = i;
    hi = p.pairs + i;
  } else {
    lo = p.pairs + i;
    hi = p.head_dim / 2 + i;
  }
}

__device__ float warp_sum(float v) {
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// One warp a token: cosines and sines once, then head by head.
template <class T, bool kNorm>
__global__ void __launch_bounds__(32 * kWarps) rotary_kernel(const __grid_constant__ RotaryParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  if (row >= p.rows) return;
  const int64_t b = row / p.tokens, s = row % p.tokens;
  const int half = p.head_dim / 2;
  float2 u[kMaxPairs / 32];
  for (int k = 0; k < kMaxPairs / 32; k++) u[k] = unit_of(p, lane + 32 * k, b, s);
  for (int h = 0; h < p.q_heads + p.k_heads; h++) {
    const bool is_k = h >= p.q_heads;
    const Heads& in = is_k ? p.k : p.q;
    const Heads& out = is_k ? p.k_out : p.q_out;
    const int head = is_k ? h - p.q_heads : h;
    const T* x = reinterpret_cast<const T*>(in.data) + b * in.batch + s * in.token + head * in.head;
    T* y = reinterpret_cast<T*>(out.data) + b * out.batch + s * out.token + head * out.head;
    const void* w = is_k ? p.k_weight : p.q_weight;
    float a[kMaxPairs / 32], c[kMaxPairs / 32], sum = 0;
    for (int k = 0; k < kMaxPairs / 32; k++) {
      const int i = lane + 32 * k;
      a[k] = c[k] = 0;
      if (i < half) {
        int lo, hi;
        elements_of(p, i, lo, hi);
        a[k] = to_float(x[lo]);
        c[k] = to_float(x[hi]);
        sum += a[k] * a[k] + c[k] * c[k];
      }
    }
    float r = 1;
    if (kNorm) r = rsqrtf(warp_sum(sum) / p.head_dim + p.eps);
    for (int k = 0; k < kMaxPairs / 32; k++) {
      const int i = lane + 32 * k;
      if (i < half) {
        int lo, hi;
        elements_of(p, i, lo, hi);
        float f = a[k], g = c[k];
        if (kNorm) {
          f = f * r * weight_at(w, p.weight_dtype, lo);
          g = g * r * weight_at(w, p.weight_dtype, hi);
        }
        y[lo] = from_float<T>(f * u[k].x - g * u[k].y);
        y[hi] = from_float<T>(g * u[k].x + f * u[k].y);
      }
    }
  }
}

template <class T>
__global__ void __launch_bounds__(32 * kWarps) norm_rotary_backward_kernel(const __grid_constant__ RotaryParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int half = p.head_dim / 2;
  float dw[2][2][kMaxPairs / 32] = {};   // q, k; low, high
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp; row < p.rows; row += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t b = row / p.tokens, s = row % p.tokens;
    float2 u[kMaxPairs / 32];
    for (int k = 0; k < kMaxPairs / 32; k++) u[k] = unit_of(p, lane + 32 * k, b, s);
    for (int t = 0; t < 2; t++) {
      const Heads& in = t ? p.k : p.q;
      const Heads& gr = t ? p.k_grad : p.q_grad;
      const Heads& out = t ? p.k_out : p.q_out;
      const void* w = t ? p.k_weight : p.q_weight;
      for (int h = 0; h < (t ? p.k_heads : p.q_heads); h++) {
        const T* x = reinterpret_cast<const T*>(in.data) + b * in.batch + s * in.token + h * in.head;
        const T* dy = reinterpret_cast<const T*>(gr.data) + b * gr.batch + s * gr.token + h * gr.head;
        T* dx = reinterpret_cast<T*>(out.data) + b * out.batch + s * out.token + h * out.head;
        float a[kMaxPairs / 32][2], g[kMaxPairs / 32][2], v[kMaxPairs / 32][2], sum = 0, dot = 0;
        for (int k = 0; k < kMaxPairs / 32; k++) {
          const int i = lane + 32 * k;
          a[k][0] = a[k][1] = g[k][0] = g[k][1] = v[k][0] = v[k][1] = 0;
          if (i < half) {
            int lo, hi;
            elements_of(p, i, lo, hi);
            a[k][0] = to_float(x[lo]);
            a[k][1] = to_float(x[hi]);
            const float e = to_float(dy[lo]), f = to_float(dy[hi]);
            g[k][0] = e * u[k].x - f * u[k].y;
            g[k][1] = f * u[k].x + e * u[k].y;
            v[k][0] = weight_at(w, p.weight_dtype, lo);
            v[k][1] = weight_at(w, p.weight_dtype, hi);
            sum += a[k][0] * a[k][0] + a[k][1] * a[k][1];
            dot += g[k][0] * v[k][0] * a[k][0] + g[k][1] * v[k][1] * a[k][1];
          }
        }
        const float r = rsqrtf(warp_sum(sum) / p.head_dim + p.eps);
        const float m = warp_sum(dot) * r / p.head_dim;   // mean(g w n)
        for (int k = 0; k < kMaxPairs / 32; k++) {
          const int i = lane + 32 * k;
          if (i < half) {
            int at[2];
            elements_of(p, i, at[0], at[1]);
            for (int e = 0; e < 2; e++) {
              const float n = a[k][e] * r;
              dx[at[e]] = from_float<T>(r * (g[k][e] * v[k][e] - n * m));
              dw[t][e][k] += g[k][e] * n;
            }
          }
        }
      }
    }
  }
  __shared__ float part[kWarps][2 * kMaxPairs];
  for (int t = 0; t < 2; t++) {
    for (int k = 0; k < kMaxPairs / 32; k++) {
      const int i = lane + 32 * k;
      if (i < half) {
        int lo, hi;
        elements_of(p, i, lo, hi);
        part[warp][lo] = dw[t][0][k];
        part[warp][hi] = dw[t][1][k];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.head_dim; i += 32 * kWarps) {
      float sum = 0;
      for (int w = 0; w < kWarps; w++) sum += part[w][i];
      p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + t) * p.head_dim + i] = sum;
    }
    __syncthreads();
  }
}

__global__ void weight_grad_kernel(const float* partial, int blocks, int head_dim, int dtype, void* q, void* k) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= 2 * head_dim) return;
  float sum = 0;
  for (int b = 0; b < blocks; b++) sum += partial[static_cast<int64_t>(b) * 2 * head_dim + i];
  void* out = i < head_dim ? q : k;
  const int at = i % head_dim;
  if (!out) return;
  if (dtype == MLXD_F32) static_cast<float*>(out)[at] = sum;
  else if (dtype == MLXD_F16) static_cast<__half*>(out)[at] = __float2half_rn(sum);
  else static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(sum);
}

Heads heads_of(const mlxd_heads& h) {
  return Heads{static_cast<char*>(h.data), h.stride_batch, h.stride_token, h.stride_head};
}

bool absent(const mlxd_heads& h) {
  return h.data == nullptr;
}

int backward_blocks(int64_t rows, int sms) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + kWarps - 1) / kWarps, 4 * sms)));
}

enum class Pass { kRotary, kNorm, kBackward };

int check_sizes(const char* entry, const mlxd_rotary_desc* d) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  if (!d) return bad("no descriptor");
  if (d->dtype != MLXD_F32 && d->dtype != MLXD_BF16 && d->dtype != MLXD_F16) return bad("tensors must be float32, bfloat16 or float16");
  if (d->batch < 0 || d->tokens < 0 || d->q_heads < 0 || d->k_heads < 0) return bad("negative size");
  if (d->head_dim <= 0 || d->head_dim % 2 || d->head_dim > MLXD_ROTARY_MAX_HEAD_DIM) {
    return bad("head_dim must be even, from 2 to " + std::to_string(MLXD_ROTARY_MAX_HEAD_DIM) + " (got " + std::to_string(d->head_dim) + ")");
  }
  return MLXD_OK;
}

int params_of(const char* entry, const mlxd_rotary_desc* d, Pass pass, RotaryParams& p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  const int rc = check_sizes(entry, d);
  if (rc != MLXD_OK) return rc;
  std::memset(&p, 0, sizeof(p));
  if (d->n_axes < 1 || d->n_axes > MLXD_ROTARY_MAX_AXES) return bad("1 to " + std::to_string(MLXD_ROTARY_MAX_AXES) + " axes");
  int64_t pairs = 0;
  int left[MLXD_ROTARY_MAX_AXES];
  for (int a = 0; a < d->n_axes; a++) {
    if (d->sections[a] < 0) return bad("negative section");
    pairs += left[a] = d->sections[a];
  }
  if (pairs < 1 || 2 * pairs > d->head_dim) {
    return bad("sections hold " + std::to_string(pairs) + " pairs, a head of " + std::to_string(d->head_dim) + " has 1 to " + std::to_string(d->head_dim / 2));
  }
  for (int i = 0, a = 0; i < pairs; i++) {
    if (d->interleaved) {
      while (!left[a]) a = (a + 1) % d->n_axes;
    } else {
      while (!left[a]) a++;
    }
    p.axes[i >> 4] |= static_cast<uint32_t>(a) << (2 * (i & 15));
    left[a]--;
    if (d->interleaved) a = (a + 1) % d->n_axes;
  }
  if (d->positions_dtype != MLXD_I32 && d->positions_dtype != MLXD_I64 && d->positions_dtype != MLXD_F32) {
    return bad("positions must be int32, int64 or float32");
  }
  if (pass != Pass::kRotary) {
    if (d->weight_dtype != MLXD_F32 && d->weight_dtype != MLXD_BF16 && d->weight_dtype != MLXD_F16) {
      return bad("weights must be float32, bfloat16 or float16");
    }
    if (!(d->eps >= 0)) return bad("eps must not be negative");
  }
  const bool work = d->batch && d->tokens && (d->q_heads || d->k_heads);
  if (work) {
    if (!d->positions || !d->frequencies) return bad("positions and frequencies are needed");
    if (d->q_heads && (absent(d->q) || absent(d->q_out))) return bad("q and q_out are needed");
    if (d->k_heads && (absent(d->k) || absent(d->k_out))) return bad("k and k_out are needed");
    if (pass == Pass::kBackward && ((d->q_heads && absent(d->q_grad)) || (d->k_heads && absent(d->k_grad)))) return bad("q_grad and k_grad are needed");
  }
  p.q = heads_of(d->q);
  p.k = heads_of(d->k);
  p.q_out = heads_of(d->q_out);
  p.k_out = heads_of(d->k_out);
  p.q_grad = heads_of(d->q_grad);
  p.k_grad = heads_of(d->k_grad);
  p.positions = d->positions;
  p.pos_axis = d->positions_stride_axis;
  p.pos_batch = d->positions_stride_batch;
  p.pos_token = d->positions_stride_token;
  p.frequencies = d->frequencies;
  p.q_weight = d->q_weight;
  p.k_weight = d->k_weight;
  p.rows = static_cast<int64_t>(d->batch) * d->tokens;
  p.tokens = d->tokens;
  p.q_heads = d->q_heads;
  p.k_heads = d->k_heads;
  p.head_dim = d->head_dim;
  p.pairs = static_cast<int>(pairs);
  p.positions_dtype = d->positions_dtype;
  p.weight_dtype = d->weight_dtype;
  p.adjacent = d->adjacent ? 1 : 0;
  // the backward pass turns the gradient back
  p.sign = (d->inverse != 0) != (pass == Pass::kBackward) ? -1.0f : 1.0f;
  p.eps = d->eps;
  return MLXD_OK;
}

template <bool kNorm>
cudaError_t launch_forward(const RotaryParams& p, int dtype, cudaStream_t stream) {
  const int64_t blocks = (p.rows + kWarps - 1) / kWarps;
  const dim3 grid(static_cast<unsigned>(blocks)), block(32 * kWarps);
  if (dtype == MLXD_F32) rotary_kernel<float, kNorm><<<grid, block, 0, stream>>>(p);
  else if (dtype == MLXD_F16) rotary_kernel<__half, kNorm><<<grid, block, 0, stream>>>(p);
  else rotary_kernel<__nv_bfloat16, kNorm><<<grid, block, 0, stream>>>(p);
  return cudaGetLastError();
}

int forward(const char* entry, int device, void* stream, const mlxd_rotary_desc* d, Pass pass) {
  RotaryParams p;
  const int rc = params_of(entry, d, pass, p);
  if (rc != MLXD_OK) return rc;
  if (!p.rows || !(p.q_heads + p.k_heads)) return MLXD_OK;
  if (p.rows > (int64_t{1} << 31)) return fail(MLXD_ERR_INVALID, std::string(entry) + ": more than 2^31 tokens");
  MLXD_ON_DEVICE(device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = pass == Pass::kNorm ? launch_forward<true>(p, d->dtype, s) : launch_forward<false>(p, d->dtype, s);
  return e == cudaSuccess ? MLXD_OK : fail_cuda(e, entry);
}

}  // namespace

int device_sms(int device, int* sms) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];
  if (device < 0 || device >= kDevices) return fail(MLXD_ERR_INVALID, "device index out of range");
  *sms = known[device].load(std::memory_order_relaxed);
  if (!*sms) {
    MLXD_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
    known[device].store(*sms, std::memory_order_relaxed);
  }
  return MLXD_OK;
}

}  // namespace mlxd

using namespace mlxd;

extern "C" int mlxd_rotary(int device, void* cuda_stream, const mlxd_rotary_desc* d) {
  return guarded("rotary", [&] { return forward("rotary", device, cuda_stream, d, Pass::kRotary); });
}

extern "C" int mlxd_qk_norm_rotary(int device, void* cuda_stream, const mlxd_rotary_desc* d) {
  return guarded("qk_norm_rotary", [&] { return forward("qk_norm_rotary", device, cuda_stream, d, Pass::kNorm); });
}

extern "C" int mlxd_qk_norm_rotary_workspace(int device, const mlxd_rotary_desc* d, size_t* bytes) {
  return guarded("qk_norm_rotary_workspace", [&] {
    int rc = check_sizes("qk_norm_rotary_workspace", d);
    if (rc != MLXD_OK) return rc;
    if (!bytes) return fail(MLXD_ERR_INVALID, "qk_norm_rotary_workspace: no place for the result");
    int sms = 0;
    rc = device_sms(device, &sms);
    if (rc != MLXD_OK) return rc;
    *bytes = sizeof(float) * 2 * d->head_dim * backward_blocks(static_cast<int64_t>(d->batch) * d->tokens, sms);
    return static_cast<int>(MLXD_OK);
  });
}

extern "C" int mlxd_qk_norm_rotary_backward(int device, void* cuda_stream, const mlxd_rotary_desc* d) {
  return guarded("qk_norm_rotary_backward", [&] {
    const char* entry = "qk_norm_rotary_backward";
    RotaryParams p;
    int rc = params_of(entry, d, Pass::kBackward, p);
    if (rc != MLXD_OK) return rc;
    if ((d->q_weight != nullptr) != (d->q_weight_grad != nullptr) || (d->k_weight != nullptr) != (d->k_weight_grad != nullptr)) {
      return fail(MLXD_ERR_INVALID, std::string(entry) + ": a weight and its gradient come together");
    }
    if (p.rows > (int64_t{1} << 31)) return fail(MLXD_ERR_INVALID, std::string(entry) + ": more than 2^31 tokens");
    int sms = 0;
    rc = device_sms(device, &sms);
    if (rc != MLXD_OK) return rc;
    const int blocks = backward_blocks(p.rows, sms);
    if (!d->workspace || d->workspace_bytes < sizeof(float) * 2 * d->head_dim * blocks) {
      return fail(MLXD_ERR_INVALID, std::string(entry) + ": workspace too small");
    }
    p.partial = static_cast<float*>(d->workspace);
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (d->dtype == MLXD_F32) norm_rotary_backward_kernel<float><<<blocks, 32 * kWarps, 0, s>>>(p);
    else if (d->dtype == MLXD_F16) norm_rotary_backward_kernel<__half><<<blocks, 32 * kWarps, 0, s>>>(p);
    else norm_rotary_backward_kernel<__nv_bfloat16><<<blocks, 32 * kWarps, 0, s>>>(p);
    MLXD_CUDA(cudaGetLastError());
    if (d->q_weight_grad || d->k_weight_grad) {
      weight_grad_kernel<<<(2 * d->head_dim + 127) / 128, 128, 0, s>>>(p.partial, blocks, d->head_dim, d->weight_dtype, d->q_weight_grad, d->k_weight_grad);
      MLXD_CUDA(cudaGetLastError());
    }
    return static_cast<int>(MLXD_OK);
  });
}
