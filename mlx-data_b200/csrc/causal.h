// What the parts of cached and window attention share: queries that read the keys at places before theirs.
#pragma once

#include "cache.h"
#include "cross.h"

namespace mlxd {

struct CausalParams {
  Heads q, k, v, out, dout, dq, dk, dv;   // k, v of a cache: batch is the page, token the row
  float* lse;
  const float* lse_grad;        // backward: the gradient of lse, or null
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

// How rows lie in tiles of 128: the tokens of a key head's query heads, head by head within a token.
struct RowTiles {
  int heads, tokens;            // of a tile
  int chunks;                   // of a key head's query heads, where they are more than a tile has rows
  int tiles;                    // of a sample, chunk by chunk
};

inline RowTiles row_tiles(const CausalParams& p) {
  RowTiles r;
  r.heads = p.group < 128 ? p.group : 128;
  r.tokens = 128 / r.heads;
  r.chunks = (p.group + r.heads - 1) / r.heads;
  r.tiles = (p.tokens + r.tokens - 1) / r.tokens;
  return r;
}

// CTAs of an SM in the kernel for few rows: eight rows a block.
constexpr int step_ctas(int dim, int blocks) { return dim > 64 ? (blocks == 1 ? 3 : 2) : (blocks == 1 ? 4 : 3); }

struct ForwardParams {
  CausalParams p;
  RowTiles rows;
  int splits;                   // of a sample's keys
  int steps;                    // few rows, by the kernel for these:
  int cluster;                  // so many CTAs share a split's keys and join what they have
  int halves;                   // else: a CTA has one tile of rows, whose keys its two halves take tile by tile in turns
  int parts;                    // splits * (halves ? 2 : 1); 1: results are final
  float* part_out;              // [parts][batch, q_heads, tokens][head_dim]
  float* part_lse;              // [parts][batch, q_heads, tokens]
};

struct CausalMaps {
  CUtensorMap q, k, v, dout;   // forward: the first three
};

// Splits and parts of a call, but for where the parts lie.
ForwardParams forward_plan(const CausalParams& p, bool paged, int sms);
size_t forward_workspace(const ForwardParams& f);
cudaError_t launch_causal_step(const ForwardParams& f, int dtype, cudaStream_t stream);
cudaError_t launch_causal_join(const ForwardParams& f, int dtype, cudaStream_t stream);
cudaError_t launch_causal_forward(const ForwardParams& f, const CausalMaps& maps, bool paged, int dtype, cudaStream_t stream);
size_t backward_workspace(const CausalParams& p);
cudaError_t launch_causal_backward(const CausalParams& p, void* workspace, const CausalMaps& maps, int dtype, cudaStream_t stream);

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

// Bits `from` to `to` - 1 of the 64 that begin at `first`.
__device__ __forceinline__ uint64_t bits_of(int first, int from, int to) {
  const int lo = max(from - first, 0), hi = min(to - first, 64);
  return lo < hi ? (~uint64_t{0} >> (64 - (hi - lo))) << lo : 0;
}

// 16 packed elements of a row, 32 bytes: one store where they start on such a boundary, so that whole sectors are written.
__device__ __forceinline__ void store_row_part(void* to, const uint32_t (&v)[8], int units) {
  if (units >= 2 && reinterpret_cast<uintptr_t>(to) % 32 == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 : : "l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
    return;
  }
  if (units >= 1) *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
  if (units >= 2) *(reinterpret_cast<uint4*>(to) + 1) = make_uint4(v[4], v[5], v[6], v[7]);
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
