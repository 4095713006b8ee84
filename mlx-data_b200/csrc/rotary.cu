// Rotary positions with several axes, alone or behind a norm of every head, forward and backward.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

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
  float* partial;               // [blocks][head_dim] sums of the weights' gradients
  int64_t rows;                 // batch * tokens
  int tokens, q_heads, k_heads, head_dim, pairs;
  int positions_dtype, weight_dtype, adjacent;
  float sign, eps;              // sign: -1 turns back
  int lanes;                    // of a warp for one head, a power of two
  int parts, part_heads;        // forward: a token's heads are cut into so many parts
  int q_blocks;                 // backward: CTAs that take queries
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

// How a warp lies over a head.  A lane owns units of kV pairs: two vectors of kV elements (the low and the high elements of its
// pairs, or, where pairs are neighbours, 2 kV elements in a row).  kL lanes cover a head, so a warp takes 32 / kL heads at once;
// kUnits > 1 only where a lane takes single pairs (kV == 1) of a head of more than 64 elements.
template <class T, int kV>
struct alignas(sizeof(T) * kV) Vec {
  T v[kV];
};

template <class T, int kV, int kUnits, bool kAdjacent>
struct Lane {
  int at[kUnits][2];            // first elements of the two vectors
  bool owns[kUnits];
  float2 turn[kUnits * kV];     // cos, sin of the pairs

  __device__ Lane(const RotaryParams& p, int first) {
    for (int k = 0; k < kUnits; k++) {
      const int i = (first + 32 * k) * kV;   // kUnits > 1: 32 lanes a head
      owns[k] = i < p.head_dim / 2;
      if (kAdjacent) {
        at[k][0] = 2 * i;
        at[k][1] = 2 * i + kV;
      } else {
        int lo, hi;
        elements_of(p, i, lo, hi);
        at[k][0] = lo;
        at[k][1] = hi;
      }
    }
  }

  // The warp works out each angle of its token once, in `table`, and every lane takes those of its pairs.
  __device__ void angles(const RotaryParams& p, int lane, int first, uint32_t row, float2* table) {
    const uint32_t b = row / p.tokens, s = row - b * p.tokens;
    for (int i = lane; i < p.head_dim / 2; i += 32) table[i] = unit_of(p, i, b, s);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
#pragma unroll
      for (int j = 0; j < kV; j++) turn[k * kV + j] = owns[k] ? table[(first + 32 * k) * kV + j] : make_float2(1.0f, 0.0f);
    }
    __syncwarp();
  }

  struct Raw {
    Vec<T, kV> v[kUnits][2];
  };

  __device__ void load(const T* x, bool there, Raw& r) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if (owns[k] && there) {
        r.v[k][0] = *reinterpret_cast<const Vec<T, kV>*>(x + at[k][0]);
        r.v[k][1] = *reinterpret_cast<const Vec<T, kV>*>(x + at[k][1]);
      }
    }
  }

  __device__ void widen(const Raw& r, float (&e)[kUnits][2 * kV]) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
#pragma unroll
      for (int j = 0; j < kV; j++) {
        e[k][j] = owns[k] ? to_float(r.v[k][0].v[j]) : 0.0f;
        e[k][kV + j] = owns[k] ? to_float(r.v[k][1].v[j]) : 0.0f;
      }
    }
  }

  __device__ void store(T* x, const float (&e)[kUnits][2 * kV]) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if (!owns[k]) continue;
      Vec<T, kV> v[2];
#pragma unroll
      for (int j = 0; j < kV; j++) {
        v[0].v[j] = from_float<T>(e[k][j]);
        v[1].v[j] = from_float<T>(e[k][kV + j]);
      }
      *reinterpret_cast<Vec<T, kV>*>(x + at[k][0]) = v[0];
      *reinterpret_cast<Vec<T, kV>*>(x + at[k][1]) = v[1];
    }
  }

  __device__ void turned(float (&e)[kUnits][2 * kV]) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
#pragma unroll
      for (int j = 0; j < kV; j++) {
        const int lo = kAdjacent ? 2 * j : j, hi = kAdjacent ? 2 * j + 1 : kV + j;
        const float2 u = turn[k * kV + j];
        const float a = e[k][lo], b = e[k][hi];
        e[k][lo] = a * u.x - b * u.y;
        e[k][hi] = b * u.x + a * u.y;
      }
    }
  }

  __device__ void weights(const void* w, int dtype, float (&e)[kUnits][2 * kV]) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
#pragma unroll
      for (int j = 0; j < kV; j++) {
        e[k][j] = owns[k] ? weight_at(w, dtype, at[k][0] + j) : 0.0f;
        e[k][kV + j] = owns[k] ? weight_at(w, dtype, at[k][1] + j) : 0.0f;
      }
    }
  }
};

__device__ float lanes_sum(float v, int lanes) {
  for (int d = lanes >> 1; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// One warp a token, or a part of its heads where tokens are few: cosines and sines once, then its heads, 32 / lanes at a time.
// The next heads are loaded while these are worked on.
template <class T, int kV, int kUnits, bool kAdjacent, bool kNorm>
__global__ void __launch_bounds__(32 * kWarps) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float2 table[kWarps][kMaxPairs];
  const int lane = threadIdx.x & 31, first = lane & (p.lanes - 1), warp = threadIdx.x / 32;
  const uint32_t item = blockIdx.x * kWarps + warp;
  const uint32_t row = item / p.parts, part = item - row * p.parts;
  if (row >= p.rows) return;
  const int64_t b = row / static_cast<uint32_t>(p.tokens), s = row - b * p.tokens;
  Lane<T, kV, kUnits, kAdjacent> me(p, first);
  const int step = 32 / p.lanes;
  const int heads = p.q_heads + p.k_heads, end = min(heads, static_cast<int>(part + 1) * p.part_heads);
  const auto source = [&](int h) {
    const bool is_k = h >= p.q_heads;
    const Heads& x = is_k ? p.k : p.q;
    return reinterpret_cast<const T*>(x.data) + b * x.batch + s * x.token + (is_k ? h - p.q_heads : h) * x.head;
  };
  typename Lane<T, kV, kUnits, kAdjacent>::Raw raw;
  int h = part * p.part_heads + lane / p.lanes;
  me.load(source(h), h < end, raw);
  me.angles(p, lane, first, row, table[warp]);
  float w[kUnits][2 * kV];
  int held = -1;   // whose weights are in w
  for (int base = part * p.part_heads; base < end; base += step, h += step) {
    float e[kUnits][2 * kV];
    me.widen(raw, e);
    const bool is_k = h >= p.q_heads;
    me.load(source(h + step), h + step < end, raw);
    if (kNorm) {
      if (held != is_k) me.weights(is_k ? p.k_weight : p.q_weight, p.weight_dtype, w);
      held = is_k;
      float sum = 0;
#pragma unroll
      for (int k = 0; k < kUnits; k++) {
#pragma unroll
        for (int j = 0; j < 2 * kV; j++) sum += e[k][j] * e[k][j];
      }
      const float r = rsqrtf(lanes_sum(sum, p.lanes) / p.head_dim + p.eps);
#pragma unroll
      for (int k = 0; k < kUnits; k++) {
#pragma unroll
        for (int j = 0; j < 2 * kV; j++) e[k][j] *= r * w[k][j];
      }
    }
    me.turned(e);
    if (h < end) {
      const Heads& y = is_k ? p.k_out : p.q_out;
      me.store(reinterpret_cast<T*>(y.data) + b * y.batch + s * y.token + (is_k ? h - p.q_heads : h) * y.head, e);
    }
  }
}

// The first p.q_blocks CTAs take the tokens' queries, the others their keys, so that a lane holds the sums of one weight's
// gradient: over all tokens it meets, then over the lanes and warps of the CTA in a fixed order, one row of p.partial a CTA.
template <class T, int kV, int kUnits, bool kAdjacent>
__global__ void __launch_bounds__(32 * kWarps, 4) norm_rotary_backward_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float2 table[kWarps][kMaxPairs];
  const int lane = threadIdx.x & 31, first = lane & (p.lanes - 1), warp = threadIdx.x / 32;
  const bool is_k = static_cast<int>(blockIdx.x) >= p.q_blocks;
  const Heads& in = is_k ? p.k : p.q;
  const Heads& gr = is_k ? p.k_grad : p.q_grad;
  const Heads& out = is_k ? p.k_out : p.q_out;
  const int heads = is_k ? p.k_heads : p.q_heads;
  const uint32_t block = is_k ? blockIdx.x - p.q_blocks : blockIdx.x;
  const uint32_t stride = (is_k ? gridDim.x - p.q_blocks : p.q_blocks) * kWarps;
  Lane<T, kV, kUnits, kAdjacent> me(p, first);
  const int step = 32 / p.lanes;
  float w[kUnits][2 * kV], dw[kUnits][2 * kV] = {};
  me.weights(is_k ? p.k_weight : p.q_weight, p.weight_dtype, w);
  for (uint32_t row = block * kWarps + warp; row < p.rows; row += stride) {
    const int64_t b = row / static_cast<uint32_t>(p.tokens), s = row - b * p.tokens;
    const T* x = reinterpret_cast<const T*>(in.data) + b * in.batch + s * in.token;
    const T* dy = reinterpret_cast<const T*>(gr.data) + b * gr.batch + s * gr.token;
    T* dx = reinterpret_cast<T*>(out.data) + b * out.batch + s * out.token;
    typename Lane<T, kV, kUnits, kAdjacent>::Raw rx, rg;
    int h = lane / p.lanes;
    me.load(x + h * in.head, h < heads, rx);
    me.load(dy + h * gr.head, h < heads, rg);
    me.angles(p, lane, first, row, table[warp]);
    for (int base = 0; base < heads; base += step, h += step) {
      float e[kUnits][2 * kV], g[kUnits][2 * kV];
      me.widen(rx, e);
      me.widen(rg, g);
      me.load(x + (h + step) * in.head, h + step < heads, rx);
      me.load(dy + (h + step) * gr.head, h + step < heads, rg);
      me.turned(g);
      float sum = 0, dot = 0;
#pragma unroll
      for (int k = 0; k < kUnits; k++) {
#pragma unroll
        for (int j = 0; j < 2 * kV; j++) {
          sum += e[k][j] * e[k][j];
          dot += g[k][j] * w[k][j] * e[k][j];
        }
      }
      const float r = rsqrtf(lanes_sum(sum, p.lanes) / p.head_dim + p.eps);
      const float m = lanes_sum(dot, p.lanes) * r / p.head_dim;   // mean(g w n)
      if (h < heads) {
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
#pragma unroll
          for (int j = 0; j < 2 * kV; j++) {
            const float n = e[k][j] * r;
            dw[k][j] += g[k][j] * n;
            e[k][j] = r * (g[k][j] * w[k][j] - n * m);
          }
        }
        me.store(dx + h * out.head, e);
      }
    }
  }
  if (is_k ? !p.k_weight : !p.q_weight) return;
  // lanes that hold the same elements of other heads, then the warps
#pragma unroll
  for (int k = 0; k < kUnits; k++) {
#pragma unroll
    for (int j = 0; j < 2 * kV; j++) {
      for (int d = p.lanes; d < 32; d <<= 1) dw[k][j] += __shfl_xor_sync(~0u, dw[k][j], d);
    }
  }
  float* part = reinterpret_cast<float*>(table[warp]);   // head_dim values fit: 2 * kMaxPairs
  __syncwarp();
  if (lane < p.lanes) {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if (!me.owns[k]) continue;
#pragma unroll
      for (int j = 0; j < kV; j++) {
        part[me.at[k][0] + j] = dw[k][j];
        part[me.at[k][1] + j] = dw[k][kV + j];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.head_dim; i += 32 * kWarps) {
    float sum = 0;
    for (int v = 0; v < kWarps; v++) sum += reinterpret_cast<const float*>(table[v])[i];
    p.partial[static_cast<int64_t>(blockIdx.x) * p.head_dim + i] = sum;
  }
}

// Sums of the CTAs' rows, 32 elements a CTA: warp r takes rows r, r + 32, ..., then the warps are summed in order.
__global__ void __launch_bounds__(1024) weight_grad_kernel(const __grid_constant__ RotaryParams p, int blocks, void* dq, void* dk) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, at = blockIdx.x * 32 + lane;
  const bool is_k = blockIdx.y;
  const int from = is_k ? p.q_blocks : 0, to = is_k ? blocks : p.q_blocks;
  void* out = is_k ? dk : dq;
  if (!out) return;
  float sum = 0;
  if (at < p.head_dim) {
    for (int b = from + warp; b < to; b += 32) sum += p.partial[static_cast<int64_t>(b) * p.head_dim + at];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp || at >= p.head_dim) return;
  sum = 0;
  for (int w = 0; w < 32; w++) sum += sums[w][lane];
  if (p.weight_dtype == MLXD_F32) static_cast<float*>(out)[at] = sum;
  else if (p.weight_dtype == MLXD_F16) static_cast<__half*>(out)[at] = __float2half_rn(sum);
  else static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(sum);
}

Heads heads_of(const mlxd_heads& h) {
  return Heads{static_cast<char*>(h.data), h.stride_batch, h.stride_token, h.stride_head};
}

bool absent(const mlxd_heads& h) {
  return h.data == nullptr;
}

// CTAs of the backward pass: queries' and keys' in proportion to their heads, four of each SM at most.
void backward_blocks(int64_t rows, int q_heads, int k_heads, int sms, int* q_blocks, int* blocks) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>((rows + kWarps - 1) / kWarps, 4 * sms));
  const int heads = q_heads + k_heads;
  const auto share = [&](int h) { return h ? static_cast<int>(std::max<int64_t>(1, std::min(most, (4 * sms * static_cast<int64_t>(h) + heads / 2) / heads))) : 0; };
  *q_blocks = share(q_heads);
  *blocks = *q_blocks + share(k_heads);
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
  if (static_cast<int64_t>(d->batch) * d->tokens > INT32_MAX) return bad("more than 2^31 - 1 tokens");
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

// Elements of a vector: 16 bytes where every row and both vectors of a lane start on such a boundary, else 8 bytes (heads
// of 72 16-bit elements), else single elements.
int vector_of(const RotaryParams& p, int bytes, bool backward) {
  for (int v = 16 / bytes; v > 1; v = v == 8 ? 4 : 1) {
    bool fits = p.head_dim / 2 % v == 0 && (p.adjacent || p.pairs % v == 0);
    const auto rows = [&](const Heads& h, int heads) {
      if (!heads) return;
      const int64_t unit = v * bytes;
      fits = fits && reinterpret_cast<uintptr_t>(h.data) % unit == 0 && (p.rows <= p.tokens || h.batch * bytes % unit == 0) &&
             (p.tokens <= 1 || h.token * bytes % unit == 0) && (heads <= 1 || h.head * bytes % unit == 0);
    };
    rows(p.q, p.q_heads);
    rows(p.k, p.k_heads);
    rows(p.q_out, p.q_heads);
    rows(p.k_out, p.k_heads);
    if (backward) {
      rows(p.q_grad, p.q_heads);
      rows(p.k_grad, p.k_heads);
    }
    if (fits) return v;
  }
  return 1;
}

int lanes_of(int units) {
  int lanes = 1;
  while (lanes < units && lanes < 32) lanes *= 2;
  return lanes;
}

// Calls f with the instance's constants: vector length, units of a lane, neighbours as pairs.
template <class T, class F>
cudaError_t with_instance(const RotaryParams& p, int v, F&& f) {
  constexpr int kWide = 16 / sizeof(T);
  using std::integral_constant;
  const auto go = [&](auto vec, auto units) {
    return p.adjacent ? f(T(), vec, units, std::true_type()) : f(T(), vec, units, std::false_type());
  };
  if (v == kWide) return go(integral_constant<int, kWide>(), integral_constant<int, 1>());
  if (v == 4) return go(integral_constant<int, 4>(), integral_constant<int, 1>());
  return go(integral_constant<int, 1>(), integral_constant<int, kMaxPairs / 32>());
}

template <class F>
cudaError_t with_type(int dtype, const RotaryParams& p, int v, F&& f) {
  if (dtype == MLXD_F32) return with_instance<float>(p, v, f);
  if (dtype == MLXD_F16) return with_instance<__half>(p, v, f);
  return with_instance<__nv_bfloat16>(p, v, f);
}

int forward(const char* entry, int device, void* stream, const mlxd_rotary_desc* d, Pass pass) {
  RotaryParams p;
  int rc = params_of(entry, d, pass, p);
  if (rc != MLXD_OK) return rc;
  const int heads = p.q_heads + p.k_heads;
  if (!p.rows || !heads) return MLXD_OK;
  int sms = 0;
  rc = device_sms(device, &sms);
  if (rc != MLXD_OK) return rc;
  const int v = vector_of(p, dtype_bytes(d->dtype), false);
  p.lanes = lanes_of(p.head_dim / 2 / v);
  // a token's heads are shared out among warps until there are 32 warps for every SM
  const int at_once = 32 / p.lanes, groups = (heads + at_once - 1) / at_once;
  const int64_t parts = std::min<int64_t>(groups, std::max<int64_t>(1, 32 * sms / p.rows));
  p.part_heads = static_cast<int>((groups + parts - 1) / parts) * at_once;
  p.parts = (heads + p.part_heads - 1) / p.part_heads;
  MLXD_ON_DEVICE(device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = static_cast<unsigned>((p.rows * p.parts + kWarps - 1) / kWarps);
  const cudaError_t e = with_type(d->dtype, p, v, [&](auto type, auto vec, auto units, auto adjacent) {
    using T = decltype(type);
    if (pass == Pass::kNorm) rotary_kernel<T, vec(), units(), adjacent(), true><<<blocks, 32 * kWarps, 0, s>>>(p);
    else rotary_kernel<T, vec(), units(), adjacent(), false><<<blocks, 32 * kWarps, 0, s>>>(p);
    return cudaGetLastError();
  });
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
    int q_blocks = 0, blocks = 0;
    backward_blocks(static_cast<int64_t>(d->batch) * d->tokens, d->q_heads, d->k_heads, sms, &q_blocks, &blocks);
    *bytes = sizeof(float) * d->head_dim * blocks;
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
    int sms = 0, blocks = 0;
    rc = device_sms(device, &sms);
    if (rc != MLXD_OK) return rc;
    backward_blocks(p.rows, p.q_heads, p.k_heads, sms, &p.q_blocks, &blocks);
    if (!blocks) return static_cast<int>(MLXD_OK);
    if (!d->workspace || d->workspace_bytes < sizeof(float) * d->head_dim * blocks) {
      return fail(MLXD_ERR_INVALID, std::string(entry) + ": workspace too small");
    }
    p.partial = static_cast<float*>(d->workspace);
    const int v = vector_of(p, dtype_bytes(d->dtype), true);
    p.lanes = lanes_of(p.head_dim / 2 / v);
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    MLXD_CUDA(with_type(d->dtype, p, v, [&](auto type, auto vec, auto units, auto adjacent) {
      norm_rotary_backward_kernel<decltype(type), vec(), units(), adjacent()><<<blocks, 32 * kWarps, 0, s>>>(p);
      return cudaGetLastError();
    }));
    if (d->q_weight_grad || d->k_weight_grad) {
      weight_grad_kernel<<<dim3((d->head_dim + 31) / 32, 2), 1024, 0, s>>>(p, blocks, d->q_weight_grad, d->k_weight_grad);
      MLXD_CUDA(cudaGetLastError());
    }
    return static_cast<int>(MLXD_OK);
  });
}
