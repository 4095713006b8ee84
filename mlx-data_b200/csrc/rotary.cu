// Rotary positions with several axes, alone or behind a norm of every head, forward and backward.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "attention.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kWarps = 4;                                // of a CTA
constexpr int kForwardBlocks = 7;                        // CTAs of an SM: 28 warps of 72 registers
constexpr int kBackwardBlocks = 3;                       // in the backward pass, of 165 registers
constexpr int kMaxPairs = MLXD_ROTARY_MAX_HEAD_DIM / 2;
constexpr int kMaxHeads = 1 << 29;                       // of q, and of k: counts of both, and a step beyond the last, fit an int

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
  int q_rounds, k_rounds;       // forward: rounds of 32 / lanes heads of a token,
  int parts, part_rounds;       // cut into so many parts
  float inverse_dim;            // 1 / head_dim
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

// How a warp lies over a head.  A lane owns kN pairs of a head: kUnits units of kV pairs, whose elements are two vectors of kV (the low
// and the high elements of its pairs, or, where pairs are neighbours, 2 kV elements in a row).  p.lanes lanes cover a head, so a
// warp takes 32 / lanes heads at once; kUnits > 1 only where a lane takes single pairs (kV == 1) of a head of more than 64 elements.
// Arithmetic runs on two pairs at once (f32x2).
template <class T, int kV>
struct alignas(sizeof(T) * kV) Vec {
  T v[kV];
};

template <class T, int kV, int kUnits, bool kAdjacent>
struct Lane {
  static constexpr int kN = kV * kUnits;
  int at[kUnits][2];            // first elements of the two vectors
  bool owns[kUnits];

  struct Raw {
    Vec<T, kV> v[kUnits][2];
  };

  // Elements a and b of the lane's pairs.
  struct Pairs {
    float a[kN], b[kN];
  };

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

  // Which of the lane's pairs are turned, a bit each.
  __device__ uint32_t turned(const RotaryParams& p, int first) const {
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < kUnits; k++) bits |= ((1u << min(max(p.pairs - (first + 32 * k) * kV, 0), kV)) - 1) << (k * kV);
    return bits;
  }

  // Cosines and sines of the lane's pairs out of the warp's table.
  __device__ void angles(const float2* table, int first, Pairs& u) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
#pragma unroll
      for (int j = 0; j < kV; j++) {
        const float2 x = owns[k] ? table[(first + 32 * k) * kV + j] : make_float2(1.0f, 0.0f);
        u.a[k * kV + j] = x.x;
        u.b[k * kV + j] = x.y;
      }
    }
  }

  __device__ void load(const T* x, bool there, Raw& r) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if (owns[k] && there) {
        r.v[k][0] = *reinterpret_cast<const Vec<T, kV>*>(x + at[k][0]);
        r.v[k][1] = *reinterpret_cast<const Vec<T, kV>*>(x + at[k][1]);
      }
    }
  }

  // Where in a unit's 2 kV elements those of pair j are.
  static __device__ constexpr int low(int j) { return kAdjacent ? 2 * j : j; }
  static __device__ constexpr int high(int j) { return kAdjacent ? 2 * j + 1 : kV + j; }

  // Lanes beyond the head hold zeros: their part of `r` is zero from the beginning and never loaded.
  __device__ void widen(const Raw& r, Pairs& e) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if constexpr (sizeof(T) == 2 && kV > 1) {
#pragma unroll
        for (int i = 0; i < kV; i++) {   // words of two elements: first those of the low vector
          const float2 x = unpack2<T>(reinterpret_cast<const uint32_t*>(r.v[k])[i]);
          if (kAdjacent) {
            e.a[k * kV + i] = x.x;
            e.b[k * kV + i] = x.y;
          } else {
            float* to = i < kV / 2 ? e.a : e.b;
            to[k * kV + 2 * i % kV] = x.x;
            to[k * kV + 2 * i % kV + 1] = x.y;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kV; j++) {
          e.a[k * kV + j] = to_float(r.v[k][low(j) / kV].v[low(j) % kV]);
          e.b[k * kV + j] = to_float(r.v[k][high(j) / kV].v[high(j) % kV]);
        }
      }
    }
  }

  __device__ void store(T* x, const Pairs& e) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if (!owns[k]) continue;
      Vec<T, kV> v[2];
      if constexpr (sizeof(T) == 2 && kV > 1) {
#pragma unroll
        for (int i = 0; i < kV; i++) {
          const float* from = i < kV / 2 ? e.a : e.b;
          reinterpret_cast<uint32_t*>(v)[i] = kAdjacent ? pack2<T>(e.a[k * kV + i], e.b[k * kV + i])
                                                        : pack2<T>(from[k * kV + 2 * i % kV], from[k * kV + 2 * i % kV + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kV; j++) {
          v[low(j) / kV].v[low(j) % kV] = from_float<T>(e.a[k * kV + j]);
          v[high(j) / kV].v[high(j) % kV] = from_float<T>(e.b[k * kV + j]);
        }
      }
      *reinterpret_cast<Vec<T, kV>*>(x + at[k][0]) = v[0];
      *reinterpret_cast<Vec<T, kV>*>(x + at[k][1]) = v[1];
    }
  }

  // Values of a vector over the head (weights in shared memory) at the lane's elements.
  __device__ void gather(const float* w, Pairs& e) const {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
#pragma unroll
      for (int j = 0; j < kV; j++) {
        e.a[k * kV + j] = owns[k] ? w[at[k][low(j) / kV] + low(j) % kV] : 0.0f;
        e.b[k * kV + j] = owns[k] ? w[at[k][high(j) / kV] + high(j) % kV] : 0.0f;
      }
    }
  }
};

// Two neighbouring values of an array.
__device__ __forceinline__ float2 two(const float* v, int i) { return make_float2(v[i], v[i + 1]); }
__device__ __forceinline__ void put(float* v, int i, float2 x) {
  v[i] = x.x;
  v[i + 1] = x.y;
}
__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Which pairs of a lane are turned: all of every head; all or none of a lane's; any.
enum Turned { kAll, kLanes, kAny };

// Turns a lane's pairs where a part of the head passes through.  Elements that pass through stay as they are, bit by bit: a cosine of 1 and
// a sine of 0 would carry an infinity from one of two to the other.  kLanes: products with the cosines, which are 1, then those with
// the sines under a predicate; kAny: a choice for every element.  4 x 2048 tokens, 32 heads of 64, bfloat16, 28 and 16 pairs of 32: 12.2
// and 12.0 us by a predicate, 12.6 and 12.8 by choices (sines of 0: 11.6 and 11.2); 16 pairs of neighbours 13.4 and 11.5 (11.2); in
// float32, 19600 tokens, 48 heads of 64, neighbours, 79.5 and 81.5 us (80.0).
template <Turned kTurned, class L>
__device__ __forceinline__ void turn_part(uint32_t turned, const typename L::Pairs& u, typename L::Pairs& e) {
#pragma unroll
  for (int i = 0; i < L::kN; i += 2) {
    const float2 a = two(e.a, i), c = two(e.b, i), cos = two(u.a, i), sin = two(u.b, i);
    float2 x = mul2(a, cos), y = mul2(c, cos);
    if constexpr (kTurned == kLanes) {
      fma2_if(turned, c, neg2(sin), x);
      fma2_if(turned, a, sin, y);
    } else {
      x = fma2(c, neg2(sin), x);
      y = fma2(a, sin, y);
      const bool first = turned >> i & 1, second = turned >> (i + 1) & 1;
      x = make_float2(first ? x.x : a.x, second ? x.y : a.y);
      y = make_float2(first ? y.x : c.x, second ? y.y : c.y);
    }
    put(e.a, i, x);
    put(e.b, i, y);
  }
}

__device__ float lanes_sum(float v, int lanes) {
  for (int d = lanes >> 1; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

__device__ void read_weights(const RotaryParams& p, float (&w)[2][MLXD_ROTARY_MAX_HEAD_DIM]) {
  for (int i = threadIdx.x; i < p.head_dim; i += 32 * kWarps) {
    w[0][i] = weight_at(p.q_weight, p.weight_dtype, i);
    w[1][i] = weight_at(p.k_weight, p.weight_dtype, i);
  }
  __syncthreads();
}

// y = R(x r w), r = 1 / sqrt(mean(x^2) + eps): every value is read and written once, so memory is the floor.  One warp a token, or a part
// of its heads where tokens are few: each angle of the token once (its sine and cosine are what costs, and all heads share them),
// then its heads, 32 / lanes at a time, queries first.  The next heads are loaded while these are worked on.  A warp a token and no loop
// over tokens: CTAs that fit at once, looping, took 65 us instead of 46 (16 x 1024 tokens, 32 heads of 80), since a token's
// positions and sines are waited for one token after another then.  Seven CTAs an SM, by their registers, with the few spills that
// takes: without a limit (five) 48.0 us, six 46.0, seven 42.0, eight 42.4, nine 44.9 for those; 50.6, 50.6, 45.7 for five, six, seven
// with the norm (3 x 4099 tokens, 32 heads of 128, float16), 4.4 TB/s.  19600 tokens, 48 heads of 64, float32: 79 us, 6.1 TB/s;
// one token of 40 heads 2.8 us.  Bound by latency and the issue of instructions for 16-bit types (about 100 for four heads of 128; heads of
// 80 use five of eight lanes).
template <class T, int kV, int kUnits, bool kAdjacent, Turned kTurned, bool kNorm>
__global__ void __launch_bounds__(32 * kWarps, kForwardBlocks) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using L = Lane<T, kV, kUnits, kAdjacent>;
  __shared__ float2 tables[kWarps][kMaxPairs];
  __shared__ float weights[2][kNorm ? MLXD_ROTARY_MAX_HEAD_DIM : 1];
  const int lane = threadIdx.x & 31, first = lane & (p.lanes - 1), mine = lane / p.lanes, at_once = 32 / p.lanes;
  float2* table = tables[threadIdx.x / 32];
  const L me(p, first);
  if constexpr (kNorm) read_weights(p, weights);
  const uint32_t items = static_cast<uint32_t>(p.rows) * p.parts;
  const uint32_t item = blockIdx.x * kWarps + threadIdx.x / 32;
  if (item < items) {
    const uint32_t row = p.parts == 1 ? item : item / p.parts, part = item - row * p.parts;
    const uint32_t b = row / static_cast<uint32_t>(p.tokens), s = row - b * p.tokens;
    // rounds of a token: those of its queries, then those of its keys; this warp has `from` to `to` - 1 of them
    const int from = part * p.part_rounds, to = min(p.q_rounds + p.k_rounds, from + p.part_rounds);
    const int first_of[2] = {min(from, p.q_rounds), max(from, p.q_rounds) - p.q_rounds};
    const int last_of[2] = {min(to, p.q_rounds), max(to, p.q_rounds) - p.q_rounds};
    typename L::Raw raw = {}, keys = {};
    const auto source = [&](const Heads& x, int round) {
      return reinterpret_cast<const T*>(x.data) + b * x.batch + s * x.token + (round * at_once + mine) * x.head;
    };
    me.load(source(p.q, first_of[0]), first_of[0] < last_of[0] && first_of[0] * at_once + mine < p.q_heads, raw);
    me.load(source(p.k, first_of[1]), first_of[1] < last_of[1] && first_of[1] * at_once + mine < p.k_heads, keys);
    for (int i = lane; i < p.head_dim / 2; i += 32) table[i] = unit_of(p, i, b, s);
    __syncwarp();
    typename L::Pairs u, w;
    me.angles(table, first, u);
    const uint32_t turned = kTurned == kAll ? 0 : me.turned(p, first);
#pragma unroll 1
    for (int is_k = 0; is_k < 2; is_k++) {
      const Heads& in = is_k ? p.k : p.q;
      const Heads& out = is_k ? p.k_out : p.q_out;
      const int heads = is_k ? p.k_heads : p.q_heads, last = last_of[is_k];
      int round = first_of[is_k];
      if (round >= last) continue;
      if (is_k) raw = keys;
      if constexpr (kNorm) me.gather(weights[is_k], w);
      const T* x = source(in, round);
      T* y = reinterpret_cast<T*>(out.data) + b * out.batch + s * out.token + (round * at_once + mine) * out.head;
      const int64_t step = at_once * in.head, out_step = at_once * out.head;
#pragma unroll 1
      for (int h = round * at_once + mine; round < last; round++, h += at_once) {
        typename L::Pairs e;
        me.widen(raw, e);
        x += step;
        me.load(x, round + 1 < last && h + at_once < heads, raw);
        if constexpr (kNorm) {
          float2 sum = {};
#pragma unroll
          for (int i = 0; i < L::kN; i += 2) sum = fma2(two(e.a, i), two(e.a, i), fma2(two(e.b, i), two(e.b, i), sum));
          const float2 r = both(rsqrtf(lanes_sum(sum.x + sum.y, p.lanes) * p.inverse_dim + p.eps));
#pragma unroll
          for (int i = 0; i < L::kN; i += 2) {
            put(e.a, i, mul2(mul2(two(e.a, i), r), two(w.a, i)));
            put(e.b, i, mul2(mul2(two(e.b, i), r), two(w.b, i)));
          }
        }
        if constexpr (kTurned == kAll) {
#pragma unroll
          for (int i = 0; i < L::kN; i += 2) {
            const float2 a = two(e.a, i), c = two(e.b, i), cos = two(u.a, i), sin = two(u.b, i);
            put(e.a, i, fma2(c, neg2(sin), mul2(a, cos)));
            put(e.b, i, fma2(a, sin, mul2(c, cos)));
          }
        } else {
          turn_part<kTurned, L>(turned, u, e);
        }
        if (h < heads) me.store(y, e);
        y += out_step;
      }
    }
  }
}

// With g = R^-1(dy), n = x r: dw = sum g n, dx = r (g w - n mean(g w n)); r is worked out again, so that the forward pass keeps nothing.
// The first p.q_blocks CTAs take the tokens' queries, the others their keys, so that a lane holds the sums of one weight's
// gradient: over all tokens it meets, then over the lanes and warps of the CTA in a fixed order, one row of p.partial a CTA.
// Measured: forward and backward of 8 x 2048 tokens, 32 heads of 128, 160 us (4.2 TB/s).  Three CTAs of 165 registers an SM: four
// (128 registers, spills) took 177, 8-byte vectors, which need fewer, 215.
template <class T, int kV, int kUnits, bool kAdjacent, Turned kTurned>
__global__ void __launch_bounds__(32 * kWarps, kBackwardBlocks) norm_rotary_backward_kernel(const __grid_constant__ RotaryParams p) {
  using L = Lane<T, kV, kUnits, kAdjacent>;
  __shared__ float2 tables[kWarps][kMaxPairs];
  __shared__ float weights[2][MLXD_ROTARY_MAX_HEAD_DIM];
  const int lane = threadIdx.x & 31, first = lane & (p.lanes - 1), mine = lane / p.lanes, at_once = 32 / p.lanes;
  float2* table = tables[threadIdx.x / 32];
  asm volatile("griddepcontrol.launch_dependents;");
  const bool is_k = static_cast<int>(blockIdx.x) >= p.q_blocks;
  const Heads in = is_k ? p.k : p.q, gr = is_k ? p.k_grad : p.q_grad, out = is_k ? p.k_out : p.q_out;
  const int heads = is_k ? p.k_heads : p.q_heads;
  const uint32_t block = is_k ? blockIdx.x - p.q_blocks : blockIdx.x;
  const uint32_t stride = (is_k ? gridDim.x - p.q_blocks : p.q_blocks) * kWarps;
  const L me(p, first);
  read_weights(p, weights);
  const uint32_t turned = kTurned == kAll ? 0 : me.turned(p, first);
  typename L::Pairs w, dw = {};
  me.gather(weights[is_k], w);
  for (uint32_t row = block * kWarps + threadIdx.x / 32; row < p.rows; row += stride) {
    const uint32_t b = row / static_cast<uint32_t>(p.tokens), s = row - b * p.tokens;
    const T* x = reinterpret_cast<const T*>(in.data) + b * in.batch + s * in.token + mine * in.head;
    const T* dy = reinterpret_cast<const T*>(gr.data) + b * gr.batch + s * gr.token + mine * gr.head;
    T* dx = reinterpret_cast<T*>(out.data) + b * out.batch + s * out.token + mine * out.head;
    typename L::Raw rx = {}, rg = {};
    me.load(x, mine < heads, rx);
    me.load(dy, mine < heads, rg);
    for (int i = lane; i < p.head_dim / 2; i += 32) table[i] = unit_of(p, i, b, s);
    __syncwarp();
    typename L::Pairs u;
    me.angles(table, first, u);
    for (int h = mine; h - mine < heads; h += at_once) {
      typename L::Pairs e, g;
      me.widen(rx, e);
      me.widen(rg, g);
      x += at_once * in.head;
      dy += at_once * gr.head;
      me.load(x, h + at_once < heads, rx);
      me.load(dy, h + at_once < heads, rg);
      float2 sum = {}, dot = {};
      if constexpr (kTurned != kAll) turn_part<kTurned, L>(turned, u, g);
#pragma unroll
      for (int i = 0; i < L::kN; i += 2) {
        const float2 a = two(g.a, i), c = two(g.b, i), cos = two(u.a, i), sin = two(u.b, i), f = two(e.a, i), k = two(e.b, i);
        const float2 ga = kTurned == kAll ? fma2(c, neg2(sin), mul2(a, cos)) : a, gb = kTurned == kAll ? fma2(a, sin, mul2(c, cos)) : c;
        put(g.a, i, ga);
        put(g.b, i, gb);
        sum = fma2(f, f, fma2(k, k, sum));
        dot = fma2(mul2(ga, two(w.a, i)), f, fma2(mul2(gb, two(w.b, i)), k, dot));
      }
      const float r = rsqrtf(lanes_sum(sum.x + sum.y, p.lanes) * p.inverse_dim + p.eps);
      const float m = lanes_sum(dot.x + dot.y, p.lanes) * r * p.inverse_dim;   // mean(g w n)
      if (h < heads) {
#pragma unroll
        for (int i = 0; i < L::kN; i += 2) {   // n = x r, dw += g n, dx = r (g w - n m)
          const float2 na = mul2(two(e.a, i), both(r)), nb = mul2(two(e.b, i), both(r)), ga = two(g.a, i), gb = two(g.b, i);
          put(dw.a, i, fma2(ga, na, two(dw.a, i)));
          put(dw.b, i, fma2(gb, nb, two(dw.b, i)));
          put(e.a, i, mul2(both(r), fma2(na, both(-m), mul2(ga, two(w.a, i)))));
          put(e.b, i, mul2(both(r), fma2(nb, both(-m), mul2(gb, two(w.b, i)))));
        }
        me.store(dx, e);
      }
      dx += at_once * out.head;
    }
    __syncwarp();
  }
  if (is_k ? !p.k_weight : !p.q_weight) return;
  // lanes that hold the same elements of other heads, then the warps
#pragma unroll
  for (int i = 0; i < L::kN; i++) {
    for (int d = p.lanes; d < 32; d <<= 1) {
      dw.a[i] += __shfl_xor_sync(~0u, dw.a[i], d);
      dw.b[i] += __shfl_xor_sync(~0u, dw.b[i], d);
    }
  }
  float* part = reinterpret_cast<float*>(table);   // head_dim values fit: 2 * kMaxPairs
  if (lane < p.lanes) {
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      if (!me.owns[k]) continue;
#pragma unroll
      for (int j = 0; j < kV; j++) {
        part[me.at[k][L::low(j) / kV] + L::low(j) % kV] = dw.a[k * kV + j];
        part[me.at[k][L::high(j) / kV] + L::high(j) % kV] = dw.b[k * kV + j];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.head_dim; i += 32 * kWarps) {
    float sum = 0;
    for (int v = 0; v < kWarps; v++) sum += reinterpret_cast<const float*>(tables[v])[i];
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
  wait_for_kernels_before();
  if (at < p.head_dim) {
#pragma unroll 4
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

// CTAs of the backward pass: queries' and keys' in proportion to their heads, kBackwardBlocks of each SM at most.
void backward_blocks(int64_t rows, int q_heads, int k_heads, int sms, int* q_blocks, int* blocks) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>((rows + kWarps - 1) / kWarps, kBackwardBlocks * sms));
  const int heads = q_heads + k_heads;
  const auto share = [&](int h) { return h ? static_cast<int>(std::max<int64_t>(1, std::min(most, (kBackwardBlocks * sms * static_cast<int64_t>(h) + heads / 2) / heads))) : 0; };
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
  if (d->q_heads > kMaxHeads || d->k_heads > kMaxHeads) return bad("more than 2^29 heads");
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
  // a kernel reads and writes whole elements, and a misaligned one is a fault
  const int bytes = dtype_bytes(d->dtype);
  for (const mlxd_heads* h : {&d->q, &d->q_out, &d->k, &d->k_out, &d->q_grad, &d->k_grad}) {
    if (!on_boundary(h->data, bytes)) return bad("a tensor does not start on a multiple of its element's size");
  }
  if (!on_boundary(d->positions, dtype_bytes(d->positions_dtype)) || !on_boundary(d->frequencies, 4)) {
    return bad("positions or frequencies do not start on a multiple of their element's size");
  }
  if (pass != Pass::kRotary) {
    for (const void* w : {d->q_weight, d->k_weight, static_cast<const void*>(d->q_weight_grad), static_cast<const void*>(d->k_weight_grad)}) {
      if (!on_boundary(w, dtype_bytes(d->weight_dtype))) return bad("a weight or its gradient does not start on a multiple of its element's size");
    }
  }
  if (pass == Pass::kBackward && !on_boundary(d->workspace, 16)) return bad("workspace must start on 16 bytes");
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
  p.inverse_dim = 1.0f / d->head_dim;
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

// Calls f with the instance's constants: vector length, units of a lane, neighbours as pairs, which pairs are turned.
template <class T, class F>
cudaError_t with_instance(const RotaryParams& p, int v, F&& f) {
  constexpr int kWide = 16 / sizeof(T);
  using std::integral_constant;
  const auto go = [&](auto vec, auto units) {
    const auto part = [&](auto adjacent, auto kind) {
      return 2 * p.pairs == p.head_dim ? f(T(), vec, units, adjacent, integral_constant<Turned, kAll>()) : f(T(), vec, units, adjacent, kind);
    };
    // a vector of halves is turned or not (vector_of); neighbours may end inside one, single pairs of one lane lie apart
    using any = integral_constant<Turned, kAny>;
    using several = integral_constant<Turned, vec() == 1 ? kAny : kLanes>;
    if (!p.adjacent) return part(std::false_type(), several());
    if constexpr (sizeof(T) == 4) {
      if (p.pairs % vec() == 0) return part(std::true_type(), several());
    }
    return part(std::true_type(), any());
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
  if (!p.rows || !(p.q_heads + p.k_heads)) return MLXD_OK;
  int sms = 0;
  rc = device_sms(device, &sms);
  if (rc != MLXD_OK) return rc;
  const int v = vector_of(p, dtype_bytes(d->dtype), false);
  p.lanes = lanes_of(p.head_dim / 2 / v);
  // a token's heads are shared out among warps until there are 32 warps for every SM
  const int at_once = 32 / p.lanes;
  p.q_rounds = (p.q_heads + at_once - 1) / at_once;
  p.k_rounds = (p.k_heads + at_once - 1) / at_once;
  const int rounds = p.q_rounds + p.k_rounds;
  const int64_t parts = std::min<int64_t>(rounds, std::max<int64_t>(1, 32 * sms / p.rows));
  p.part_rounds = static_cast<int>((rounds + parts - 1) / parts);
  p.parts = (rounds + p.part_rounds - 1) / p.part_rounds;
  MLXD_ON_DEVICE(device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = static_cast<unsigned>((p.rows * p.parts + kWarps - 1) / kWarps);
  const cudaError_t e = with_type(d->dtype, p, v, [&](auto type, auto vec, auto units, auto adjacent, auto turned) {
    using T = decltype(type);
    if (pass == Pass::kNorm) rotary_kernel<T, vec(), units(), adjacent(), turned(), true><<<blocks, 32 * kWarps, 0, s>>>(p);
    else rotary_kernel<T, vec(), units(), adjacent(), turned(), false><<<blocks, 32 * kWarps, 0, s>>>(p);
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
    if (blocks && (!d->workspace || d->workspace_bytes < sizeof(float) * d->head_dim * blocks)) {
      return fail(MLXD_ERR_INVALID, std::string(entry) + ": workspace too small");
    }
    p.partial = static_cast<float*>(d->workspace);
    const int v = vector_of(p, dtype_bytes(d->dtype), true);
    p.lanes = lanes_of(p.head_dim / 2 / v);
    MLXD_ON_DEVICE(device);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (blocks) {
      MLXD_CUDA(with_type(d->dtype, p, v, [&](auto type, auto vec, auto units, auto adjacent, auto turned) {
        norm_rotary_backward_kernel<decltype(type), vec(), units(), adjacent(), turned()><<<blocks, 32 * kWarps, 0, s>>>(p);
        return cudaGetLastError();
      }));
    }
    // without heads too: the sums of nothing
    if (d->q_weight_grad || d->k_weight_grad) {
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3((d->head_dim + 31) / 32, 2);
      config.blockDim = dim3(1024);
      config.stream = s;
      cudaLaunchAttribute early = {};
      early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      early.val.programmaticStreamSerializationAllowed = 1;
      config.attrs = &early;
      config.numAttrs = 1;
      MLXD_CUDA(cudaLaunchKernelEx(&config, weight_grad_kernel, p, blocks, d->q_weight_grad, d->k_weight_grad));
    }
    return static_cast<int>(MLXD_OK);
  });
}
