// What the parts of cached and window attention share: queries that read the keys at places before theirs.
#pragma once

#include "cache.h"
#include "cross.h"

namespace mlxd {

struct CausalParams {
  Heads q, k, v, out, dout, dq, dk, dv;   // k, v of a cache: batch is the page, token the row
  float* lse;
  const float* lse_grad;        // backward: the gradient of lse, or null
  float* delta;                 // backward: [batch, q_heads, tokens]
  CacheParams cache;            // cached attention
  const uint8_t* tree;          // cached attention: null without one
  int64_t tree_batch, tree_token;
  const void* lengths;          // window attention: null where all tokens are there
  int lengths_dtype;
  int batch, tokens, q_heads, kv_heads, group, head_dim;
  int window, sinks;            // window: INT_MAX, above every place, where there is none
  float scale;
  int* status;
  int device;
};

cudaError_t launch_causal_forward(const CausalParams& p, bool paged, int dtype, cudaStream_t stream);
cudaError_t launch_causal_backward(const CausalParams& p, int dtype, cudaStream_t stream);

#ifdef __CUDACC__
// A sample: its queries are at the places held to held + fresh - 1, keys lie at 0 to end - 1.
struct Sequence {
  int held, fresh, end;
};

template <bool kPaged>
__device__ __forceinline__ Sequence sequence_of(const CausalParams& p, int b) {
  if (kPaged) {
    const int held = length_of(p.cache, b), fresh = count_of(p.cache, b, p.tokens);
    return {held, fresh, min(held + fresh, p.cache.capacity)};
  }
  int n = p.tokens;
  if (p.lengths) n = static_cast<int>(min(max(integer_at(p.lengths, p.lengths_dtype, b), int64_t{0}), static_cast<int64_t>(n)));
  return {0, n, n};
}

// What a query reads: keys below `sinks`, and those from `from` to `to` - 1; with a tree those of its row behind `to`.
struct Reach {
  int sinks, from, to;
};

__device__ __forceinline__ Reach reach_of(const CausalParams& p, const Sequence& s, int place, int to) {
  const int from = max(0, place - p.window + 1);
  return {min(min(p.sinks, to), from), min(from, to), to};
}
#endif

}  // namespace mlxd
