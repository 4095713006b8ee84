// Gradients of window attention: one kernel for queries, one for keys and values.  As in cross attention each works out the scores
// again, so that every sum has one owner and the same order in every call (no atomics, seven products of 128 x 128 x D for the five of the
// definition), and P and dS are rounded to 16 bits as operands of the products.  Rows are tokens and the query heads that share a key
// head, as in the forward pass.  First tokens that stay visible are keys of every query behind them: their tiles' rows are split among
// CTAs, whose parts a third kernel adds in order.
//
// 10 D operations a pair by the definition, 14 D here.  Measured: 8192 tokens, 32 heads on 8 of 128, window 2048, 4 first tokens: 471-484
// us for queries (tensor pipe active for 41 %), 514-519 for keys (52 %); with the forward pass, 16384 tokens: 2694-2770 us, 650 TFLOP/s by
// the definition.  Bound by shared memory and by the chain of a tile: products of 128 x 128 x 16 read 128 bytes a cycle where both
// operands lie there, so a tile of the first kernel takes 1800 cycles of it with its copies, of 2840 measured.
#include <algorithm>

#include "causal.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

// Warpgroups for what lies between the products, then warps for copies, products, helpers.  Queries: four, each row four threads'; keys: two
// of twice the registers (8192 tokens, window 2048, 32 heads on 8: queries 498 and 502 us, keys 594 and 514).
constexpr int kRowThreads = 640, kKeyThreads = 384;
constexpr int kMaskRing = 4;           // queries: tiles of keys in the ring are no more
constexpr int kRowRing = 8;            // keys: items in the ring are no more
constexpr int kSplitCtas = 1024;       // CTAs that share the rows of first tokens' tiles
constexpr float kLog2e = 1.4426950408889634f;

template <int kDim>
struct Sizes {
  static constexpr int kTile = 128 * kDim * 2;             // bytes of 128 tokens
  static constexpr int kBoxes = kDim / 64;
  static constexpr int kSlots = kDim == 128 ? 5 : 8;       // of the ring
  static constexpr int kShared = (2 + kSlots) * kTile;
};

struct BackwardParams {
  CausalParams p;
  RowTiles rows;
  float2* stats;                // [batch, kv_heads, tokens, group]: -lse log2(e) and delta of a row
  float* partial;               // [sink_parts][batch, kv_heads][sink_tiles][dk, dv][128][head_dim]
  int sink_tiles, sink_parts;   // tiles of keys whose rows are split into so many parts; 1: none is
};

// Keys or values: 128 tokens.
template <class S>
__device__ __forceinline__ void load_keys(uint32_t to, const CUtensorMap* map, int token, int head, int batch, uint32_t bar) {
  barrier_expect(bar, S::kTile);
  for (int x = 0; x < S::kBoxes; x++) tile_load(to + x * kBoxBytes, map, 64 * x, token, head, batch, bar);
}

// Queries or gradients of results: a tile of rows.
template <class S>
__device__ __forceinline__ void load_rows(uint32_t to, const CUtensorMap* map, const RowTiles& r, int chunk, int token, int kv_head, int batch, uint32_t bar) {
  barrier_expect(bar, S::kBoxes * r.heads * r.tokens * 128);
  for (int x = 0; x < S::kBoxes; x++) tile_load(to + x * kBoxBytes, map, 64 * x, chunk * r.heads, token, kv_head, batch, bar);
}

__device__ __forceinline__ void store_zeros(uint32_t at) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" : : "r"(at), "r"(0) : "memory");
}

// Elements `from` to `from` + kCount - 1 of a row of accumulators, scaled, rounded and written; zeros where the row has no sums, or nothing
// was summed at all (`none`, of the whole CTA).
template <class T, int kCount>
__device__ __forceinline__ void write_row(uint32_t tmem, T* to, int from, int dim, float by, bool there, bool sums, bool none) {
#pragma unroll
  for (int x = 0; x < kCount; x += 16) {
    uint32_t o[16], v[8] = {};
    if (!none) {
      tmem_load<16>(tmem + from + x, o);
      tmem_loaded(o);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = sums ? pack2<T>(__uint_as_float(o[2 * i]) * by, __uint_as_float(o[2 * i + 1]) * by) : 0u;
    }
    if (there) store_row_part(to + from + x, v, (dim - from - x) / 8);
  }
}

// D (+)= A B over 128 tokens: A 128 x 128 in tensor memory, 16 columns of every 32, as the four threads of a row leave it; B a tile.
__device__ __forceinline__ void product_over_quarters(uint32_t d, uint32_t a, uint32_t b, uint32_t how, bool add) {
#pragma unroll
  for (int k = 0; k < 8; k++) product_from_tmem(d, a + 32 * (k / 2) + 8 * (k % 2), b + (2048 * k >> 4), how, add || k > 0);
}

// Of a row and this thread's quarter of a tile of keys: sums of P dP and of P, over the keys that are read.  Scores and dP stay where they
// are.
__device__ __forceinline__ void row_sums(uint32_t scores_at, uint32_t dp_at, uint32_t read, bool single, float c, float base, float* sum, float* weights) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    uint32_t s[16], d[16];
    tmem_load<16>(scores_at + 16 * i, s);
    tmem_load<16>(dp_at + 16 * i, d);
    tmem_loaded(s);
    tmem_loaded(d);
#pragma unroll
    for (int k = 0; k < 16; k++) {
      if (read >> (16 * i + k) & 1) {
        // lse of the forward pass makes the one weight 1 but for a rounding
        const float w = exp2_of(fmaf(__uint_as_float(s[k]), c, base)), exact = single && w > 0 ? 1.0f : w;
        *weights += exact;
        *sum = fmaf(exact, __uint_as_float(d[k]), *sum);
      }
    }
  }
}

struct RowJob {
  int q0, chunk, kv_head, batch;
};

// The last tiles of rows first: without a window they have the most keys.
__device__ __forceinline__ RowJob row_job_of(const BackwardParams& f, int id) {
  RowJob j;
  j.kv_head = id % f.p.kv_heads;
  id /= f.p.kv_heads;
  j.batch = id % f.p.batch;
  id /= f.p.batch;
  j.chunk = id % f.rows.chunks;
  j.q0 = (f.rows.tiles - 1 - id / f.rows.chunks) * f.rows.tokens;
  return j;
}

// dQ = scale dS K for a tile of rows: S = Q K^T, P = exp(S - lse), dP = dO V^T, dS = P (dP - delta), delta = sum(dO O) - dlse.  Two sets of
// scores, so that the products of the next tile run beside the exponentials of this one.  What the other kernel needs of a row it leaves
// in the order in which that one reads it.
// O comes in rounded to 16 bits, and where few keys have weights dS is the small difference of dP and delta.  So where the keys of a tile's
// rows fit two tiles, whose P and dP are there before any dS (the second dP where dQ will be), delta = sum(P dP) / sum(P) of these:
// 255 tokens in float16, dQ off by 0.00036 of its size by O, 0.0003 so (0.00021 by the rounding of results alone).  A single key has the
// weight 1, so that its dS is 0 and no remainder of a rounding.
template <class T, int kDim>
__global__ void __launch_bounds__(kRowThreads, 1) causal_dq_kernel(const __grid_constant__ BackwardParams f, const __grid_constant__ CausalMaps maps) {
  using S = Sizes<kDim>;
  const CausalParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[2 + 2 * S::kSlots + 2 + 5 + kMaskRing + 1];
  __shared__ float delta_parts[4][128];   // of a row's four threads
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  __shared__ uint32_t progress;           // copies begun
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t q_at = smem_address(shared), do_at = q_at + S::kTile, ring_at = do_at + S::kTile;
  const uint32_t q_full = smem_address(bars), do_full = q_full + 8, full = q_full + 16, empty = full + 8 * S::kSlots,
                 s_full = empty + 8 * S::kSlots, dp_full = s_full + 16, ds_full = dp_full + 8, done = ds_full + 8, delta_full = done + 8,
                 dp2_full = delta_full + 8, landed = dp2_full + 8, ended = landed + 8 * kMaskRing;
  const RowJob job = row_job_of(f, blockIdx.x);
  const int batch = job.batch, kv_head = job.kv_head;
  if (threadIdx.x == 0) {
    failed = 0;
    progress = 0;
    for (const uint32_t bar : {q_full, do_full, s_full, s_full + 8, dp_full, dp2_full, done, ended}) barrier_init(bar, 1);
    for (const uint32_t bar : {ds_full, delta_full}) barrier_init(bar, 16);
    for (int i = 0; i < S::kSlots; i++) {
      barrier_init(full + 8 * i, 1);
      barrier_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kMaskRing; i++) barrier_init(landed + 8 * i, 1);
    barrier_init_done();
  }
  if (warp == 17) tmem_alloc<512>(smem_address(&tmem_slot));
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tmem = tmem_slot, dp_column = 256, dq_column = 384;   // scores in 0 and 128
  wait_for_kernels_before();
  // The other kernel's CTAs take the SMs that these leave.  They read the inputs before they wait for this kernel, so not ahead of here.
  asm volatile("griddepcontrol.launch_dependents;");
  const Sequence seq = sequence_of<false>(p, batch);
  // what the tile's rows read, in tiles of keys: first ones, then the window's
  const int end_token = min(job.q0 + f.rows.tokens, seq.fresh);
  const Reach all = job.q0 < end_token ? reach_of(p, seq, job.q0, end_token) : Reach{0, 0, 0};
  const int sink_tiles = (all.sinks + 127) / 128, main_first = max(all.from / 128, sink_tiles);
  const int n = sink_tiles + max((all.to + 127) / 128 - main_first, 0);
  const auto tile_of = [&](int j) { return j < sink_tiles ? j : j - sink_tiles + main_first; };
  const auto partial = [&](int j) {
    const int lo = tile_of(j) * 128, hi = lo + 128;
    return !(hi <= all.sinks || (lo >= all.from && hi <= all.to));
  };

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 16 && lane == 0 && n) {
      // -------------------------------------------------- copies: keys of tile 0, values of tile 0, keys of tile 1, ...
      load_rows<S>(q_at, &maps.q, f.rows, job.chunk, job.q0, kv_head, batch, q_full);
      load_rows<S>(do_at, &maps.dout, f.rows, job.chunk, job.q0, kv_head, batch, do_full);
      int issued = 0, r = 0;
      for (; issued < 2 * n; issued++) {
        const int slot = issued % S::kSlots, use = issued / S::kSlots, j = issued / 2;
        if (use && !barrier_wait(empty + 8 * slot, (use - 1) & 1, &failed)) break;
        // keys of a tile that is not read as a whole go by way of the mask warp
        const bool by_masks = !(issued & 1) && partial(j);
        load_keys<S>(ring_at + slot * S::kTile, issued & 1 ? &maps.v : &maps.k, tile_of(j) * 128, kv_head, batch, by_masks ? landed + 8 * (r % kMaskRing) : full + 8 * slot);
        *static_cast<volatile uint32_t*>(&progress) = issued + 1;
        r += by_masks;
      }
      if (failed) {   // what is under way still lands before the CTA ends
        for (int i = 0; i < kWaitTries && !(barrier_try(q_full, 0) && barrier_try(do_full, 0)); i++) {}
        r = 0;
        for (int k = 0; k < issued; k++) {
          const bool by_masks = !(k & 1) && partial(k / 2);
          const uint32_t bar = by_masks ? landed + 8 * (r % kMaskRing) : full + 8 * (k % S::kSlots), parity = (by_masks ? r / kMaskRing : k / S::kSlots) & 1;
          r += by_masks;
          if (k < issued - S::kSlots) continue;
          for (int i = 0; i < kWaitTries && !barrier_try(bar, parity); i++) {}
        }
      }
    } else if (warp == 17 && n) {
      // -------------------------------------------------- products
      constexpr uint32_t kScores = product_descriptor<T>(128, 128, false), kResults = product_descriptor<T>(128, kDim, true);
      const int steps = (p.head_dim + 15) / 16;
      const uint32_t queries = low_half(at_address(tile_descriptor(16), q_at)), grads = low_half(at_address(tile_descriptor(16), do_at)),
                     ring = low_half(at_address(tile_descriptor(16), ring_at)), ring_tokens = low_half(at_address(tile_descriptor(kBoxBytes), ring_at));
      const auto at_slot = [&](uint32_t slot) { return slot * (S::kTile >> 4); };
      const auto scores = [&](int j, uint32_t slot) {
        product_of_tiles<kDim>(tmem + 128 * (j & 1), queries, ring + at_slot(slot), kScores, steps);
        products_done(s_full + 8 * (j & 1));
      };
      const auto dp = [&](uint32_t slot) {
        product_of_tiles<kDim>(tmem + dp_column, grads, ring + at_slot(slot), kScores, steps);
        products_done(dp_full);
        products_done(empty + 8 * slot);
      };
      bool going = warp_wait3(q_full, 0, full, 0, 0, 0, &failed);
      if (going && elected()) scores(0, 0);
      __syncwarp();
      going = going && warp_wait3(do_full, 0, full + 8, 0, 0, 0, &failed);
      if (going && elected()) dp(1);
      __syncwarp();
      going = going && (n == 1 || warp_wait(full + 16, 0, &failed));
      if (going && n > 1 && elected()) scores(1, 2);
      __syncwarp();
      if (n == 2) {
        going = going && warp_wait(full + 24, 0, &failed);
        if (going && elected()) {
          product_of_tiles<kDim>(tmem + dq_column, grads, ring + at_slot(3), kScores, steps);
          products_done(dp2_full);
        }
        __syncwarp();
        going = going && warp_wait(ds_full, 0, &failed);
        tmem_after_sync();
        if (going && elected()) {
          for (int j = 0; j < 2; j++) {
            product_over_quarters(tmem + dq_column, tmem + 128 * j, ring_tokens + at_slot(2 * j), kResults, j > 0);
          }
          products_done(done);
        }
        __syncwarp();
      }
      // one look at barriers between two groups of products: the tensor cores are not far behind the thread that issues them
      Ring<S::kSlots> k, v, next_k;          // keys of this tile, values of the next, keys of the one after
      v.next(3);
      next_k.next(4);
#pragma unroll 1
      for (int j = 0; j < n && n != 2 && going; j++) {
        going = warp_wait3(ds_full, j & 1, j + 1 < n ? full + 8 * v.slot : 0, v.phase, j + 2 < n ? full + 8 * next_k.slot : 0, next_k.phase, &failed);
        if (!going) break;
        tmem_after_sync();
        if (elected()) {
          if (j + 1 < n) dp(v.slot);
          product_over_quarters(tmem + dq_column, tmem + 128 * (j & 1), ring_tokens + at_slot(k.slot), kResults, j > 0);
          products_done(empty + 8 * k.slot);
          if (j + 2 < n) scores(j + 2, next_k.slot);   // overwrites dS of tile j after it has been read
          if (j + 1 == n) products_done(done);
        }
        __syncwarp();
        k.next(2);
        v.next(2);
        next_k.next(2);
      }
      if (!going) products_end(ended);
    } else if (warp == 18) {
      // -------------------------------------------------- masks: zeros where keys are not read by any row
      int r = 0;
      for (int j = 0; j < n; j++) {
        if (!partial(j)) continue;
        const int item = 2 * j, first = tile_of(j) * 128;
        if (!warp_wait_behind(landed + 8 * (r % kMaskRing), r / kMaskRing & 1, &failed, &progress)) break;
        const uint32_t keys = ring_at + item % S::kSlots * S::kTile;
        for (int row = lane / 8; row < 128; row += 4) {   // 8 lanes a row of 128 bytes
          const int key = first + row;
          if (key < all.sinks || (key >= all.from && key < all.to)) continue;
          for (int x = 0; x < S::kBoxes; x++) store_zeros(keys + x * kBoxBytes + row * 128 + (lane & 7) * 16);
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) barrier_arrive(full + 8 * (item % S::kSlots));
        r++;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------------------------------------------- a row belongs to four threads, one for each quarter of the keys of a tile
    const int quarter = warp / 4, row = threadIdx.x & 127;
    const int token = job.q0 + row / f.rows.heads, in_group = job.chunk * f.rows.heads + row % f.rows.heads, head = kv_head * p.group + in_group;
    const bool there = row < f.rows.heads * f.rows.tokens && token < p.tokens && in_group < p.group, reads = there && token < seq.fresh;
    const Reach mine = reads ? reach_of(p, seq, token, token + 1) : Reach{0, 0, 0};
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const float c = p.scale * kLog2e;
    const int64_t stat = (static_cast<int64_t>(batch) * p.q_heads + head) * p.tokens + token;
    // a row that reads nothing gets P = 0
    const float base = reads ? row_base(p.lse[stat]) : -INFINITY;
    float part = 0, weights = 1;
    bool going = true;
    if (n == 1 || n == 2) {
      weights = 0;
      const bool single = mine.sinks + mine.to - mine.from == 1;
      for (int j = 0; j < n && going; j++) {
        going = warp_wait(s_full + 8 * j, 0, &failed) && warp_wait(j ? dp2_full : dp_full, 0, &failed);
        if (!going) break;
        tmem_after_sync();
        const int first_key = tile_of(j) * 128 + 32 * quarter;
        const uint32_t read = static_cast<uint32_t>(bits_of(first_key, mine.from, mine.to) | bits_of(first_key, 0, mine.sinks));
        row_sums(tmem + 128 * j + 32 * quarter + lanes, tmem + (j ? dq_column : dp_column) + 32 * quarter + lanes, read, single, c, base, &part, &weights);
      }
    } else if (n) {
      // delta: a warp takes two rows at a time, 16 bytes a lane (each thread its own row: 6.7 us of a CTA's 36, at 17 tiles of keys)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int of = warp * 8 + 2 * i + lane / 16, at = lane % 16 * 8;
        const int t = job.q0 + of / f.rows.heads, g = job.chunk * f.rows.heads + of % f.rows.heads, h = kv_head * p.group + g;
        float sum = 0;
        if (of < f.rows.heads * f.rows.tokens && t < seq.fresh && g < p.group && at < p.head_dim) {
          const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.out.data) + batch * p.out.batch + t * p.out.token + h * p.out.head + at);
          const uint4 b = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.dout.data) + batch * p.dout.batch + t * p.dout.token + h * p.dout.head + at);
          const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 x = unpack2<T>(u[k]), y = unpack2<T>(v[k]);
            sum += x.x * y.x + x.y * y.y;
          }
        }
        for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if (lane % 16 == 0) delta_parts[0][of] = sum;
      }
    }
    // with few keys the sums of weights too, in the ring's last place, which these do not reach
    float(*const weight_parts)[128] = reinterpret_cast<float(*)[128]>(shared + (1 + S::kSlots) * S::kTile);
    if (n <= 2) {
      delta_parts[quarter][row] = part;
      weight_parts[quarter][row] = weights;
    }
    warp_arrive(delta_full, lane);
    going = warp_wait(delta_full, 0, &failed) && going;
    const auto of_row = [&](const float(*parts)[128]) { return (parts[0][row] + parts[1][row]) + (parts[2][row] + parts[3][row]); };
    float delta = going && reads ? delta_parts[0][row] : 0.0f;
    if (n <= 2 && going) {
      delta = of_row(delta_parts);
      weights = of_row(weight_parts);
      delta = weights == 0 ? 0.0f : delta / weights;
    }
    if (p.lse_grad && reads) delta -= p.lse_grad[stat];
    if (there && quarter == 0) {
      f.stats[((static_cast<int64_t>(batch) * p.kv_heads + kv_head) * p.tokens + token) * p.group + in_group] = make_float2(base, delta);
    }
    for (int j = 0; j < n && going; j++) {
      const uint32_t scores_at = tmem + 128 * (j & 1) + 32 * quarter + lanes;
      uint32_t s[32], d[32], packed[16];
      going = warp_wait(s_full + 8 * (j & 1), j / 2 & 1, &failed);
      if (!going) break;
      tmem_after_sync();
      tmem_load<32>(scores_at, s);
      tmem_loaded(s);
#pragma unroll
      for (int k = 0; k < 32; k += 2) {
        const float2 x = fma2(make_float2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), make_float2(c, c), make_float2(base, base));
        s[k] = __float_as_uint(exp2_of(x.x));
        s[k + 1] = __float_as_uint(exp2_of(x.y));
      }
      const int first_key = tile_of(j) * 128 + 32 * quarter;
      const uint32_t read = static_cast<uint32_t>(bits_of(first_key, mine.from, mine.to) | bits_of(first_key, 0, mine.sinks));
      const bool second = n == 2 && j == 1;
      going = second || warp_wait(dp_full, j & 1, &failed);
      if (!going) break;
      tmem_after_sync();
      tmem_load<32>(tmem + (second ? dq_column : dp_column) + 32 * quarter + lanes, d);
      tmem_loaded(d);
      if (__all_sync(~0u, read == ~0u)) {
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 x = add2(make_float2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), make_float2(-delta, -delta));
          const float2 y = mul2(x, make_float2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])));
          packed[k / 2] = pack2<T>(y.x, y.y);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float x = read >> k & 1 ? (__uint_as_float(d[k]) - delta) * __uint_as_float(s[k]) : 0.0f;
          const float y = read >> (k + 1) & 1 ? (__uint_as_float(d[k + 1]) - delta) * __uint_as_float(s[k + 1]) : 0.0f;
          packed[k / 2] = pack2<T>(x, y);
        }
      }
      tmem_store<16>(scores_at, packed);
      tmem_stored();
      tmem_before_sync();
      if (n != 2 || second) warp_arrive(ds_full, lane);
    }
    if (n && going) going = warp_wait(done, 0, &failed);
    if (going) {
      tmem_after_sync();
      T* const to = reinterpret_cast<T*>(p.dq.data) + batch * p.dq.batch + token * p.dq.token + head * p.dq.head;
      // rows behind the sequence get zeros: 0 times a key that is not a number, or infinite, has made their accumulators NaN
      write_row<T, kDim / 4>(tmem + dq_column + lanes, to, quarter * (kDim / 4), p.head_dim, p.scale, there, reads, n == 0);
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 17) tmem_free<512>(tmem);
  if (failed) {   // not a number, instead of whatever the memory held; the other kernel's results are not valid either
    const RowJob at = row_job_of(f, block_again());
    for (int i = threadIdx.x / 32; i < f.rows.tokens * f.rows.heads; i += kRowThreads / 32) {
      const int token = at.q0 + i / f.rows.heads, head = at.chunk * f.rows.heads + i % f.rows.heads;
      if (token >= p.tokens || head >= p.group) continue;
      uint16_t* to = reinterpret_cast<uint16_t*>(p.dq.data) + at.batch * p.dq.batch + token * p.dq.token + (at.kv_head * p.group + head) * p.dq.head;
      for (int e = lane; e < p.head_dim; e += 32) to[e] = 0x7fff;
      if (lane == 0) f.stats[((static_cast<int64_t>(at.batch) * p.kv_heads + at.kv_head) * p.tokens + token) * p.group + head] = make_float2(NAN, NAN);
    }
    if (threadIdx.x == 0) *p.status = 1;
  }
}

struct KeyJob {
  int tile, part, kv_head, batch;
};

// Tiles of first tokens, which have the most rows, first; then in order: without a window the first have the most.
__device__ __forceinline__ KeyJob key_job_of(const BackwardParams& f, int id) {
  KeyJob j;
  j.kv_head = id % f.p.kv_heads;
  id /= f.p.kv_heads;
  j.batch = id % f.p.batch;
  id /= f.p.batch;
  const int split = f.sink_tiles * f.sink_parts;
  j.tile = id < split ? id / f.sink_parts : id - split + f.sink_tiles;
  j.part = id < split ? id % f.sink_parts : 0;
  return j;
}

// dV = P^T dO and dK = scale dS^T Q for 128 keys, over the rows that read some of them.  Scores lie the other way round (a key a lane), so
// that P^T and dS^T are operands as they are.
template <class T, int kDim>
__global__ void __launch_bounds__(kKeyThreads, 1) causal_dkv_kernel(const __grid_constant__ BackwardParams f, const __grid_constant__ CausalMaps maps) {
  using S = Sizes<kDim>;
  const CausalParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[2 + 2 * S::kSlots + 5 + 4 + kRowRing + 1];
  __shared__ float4 stats[2][2][32];      // of the rows of a tile: -lse * log2(e), delta
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  __shared__ uint32_t progress;           // copies begun
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t k_at = smem_address(shared), v_at = k_at + S::kTile, ring_at = v_at + S::kTile;
  const uint32_t k_full = smem_address(bars), v_full = k_full + 8, full = k_full + 16, empty = full + 8 * S::kSlots,
                 s_full = empty + 8 * S::kSlots, dp_full = s_full + 8, p_full = dp_full + 8, ds_full = p_full + 8, done = ds_full + 8,
                 stats_full = done + 8, stats_empty = stats_full + 16, landed = stats_empty + 16, ended = landed + 8 * kRowRing;
  const KeyJob job = key_job_of(f, blockIdx.x);
  const int k0 = job.tile * 128, kv_head = job.kv_head, batch = job.batch, tile_rows = f.rows.tokens * f.rows.heads;
  const int length = sequence_of<false>(p, batch).fresh;

  if (threadIdx.x == 0) {
    failed = 0;
    progress = 0;
    for (const uint32_t bar : {k_full, v_full, s_full, dp_full, done, stats_full, stats_full + 8, ended}) barrier_init(bar, 1);
    for (const uint32_t bar : {p_full, ds_full, stats_empty, stats_empty + 8}) barrier_init(bar, 8);
    for (int i = 0; i < S::kSlots; i++) {
      barrier_init(full + 8 * i, 1);
      barrier_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kRowRing; i++) barrier_init(landed + 8 * i, 1);
    barrier_init_done();
  }
  // a box may have fewer rows than a tile: the others are summed over too, and no copy writes them
  for (int i = threadIdx.x; i < (128 - tile_rows) * 8 * S::kBoxes * S::kSlots; i += kKeyThreads) {
    const int box = i / ((128 - tile_rows) * 8), unit = i % ((128 - tile_rows) * 8);
    store_zeros(ring_at + box * kBoxBytes + tile_rows * 128 + unit * 16);
  }
  fence_async_proxy();
  if (warp == 9) tmem_alloc<512>(smem_address(&tmem_slot));
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tmem = tmem_slot, dp_column = 128, dv_column = 256, dk_column = 384;   // scores in 0
  // tiles of rows that read the keys, chunk by chunk: this CTA has `begin` to `begin` + n - 1 of them
  const int rows_end = k0 < p.sinks || p.window >= length ? length : min(length, k0 + 127 + p.window), first_tile = k0 / f.rows.tokens;
  const int whole = k0 < length ? ((rows_end + f.rows.tokens - 1) / f.rows.tokens - first_tile) * f.rows.chunks : 0;
  const bool split = job.tile < f.sink_tiles && f.sink_parts > 1;
  const int share = split ? (whole + f.sink_parts - 1) / f.sink_parts : whole;
  const int begin = min(job.part * share, whole), n = min(share, whole - begin);
  const auto token_of = [&](int i) { return (first_tile + (begin + i) / f.rows.chunks) * f.rows.tokens; };
  const auto chunk_of = [&](int i) { return (begin + i) % f.rows.chunks; };
  // a tile in which the sequence ends before the tensor does: rows behind it are cleared
  const auto partial = [&](int i) { return length < p.tokens && token_of(i) + f.rows.tokens > length; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 8 && lane == 0 && n) {
      // -------------------------------------------------- copies: queries of tile 0, their gradients, queries of tile 1, ...
      load_keys<S>(k_at, &maps.k, k0, kv_head, batch, k_full);
      load_keys<S>(v_at, &maps.v, k0, kv_head, batch, v_full);
      int issued = 0, r = 0;
      for (; issued < 2 * n; issued++) {
        const int slot = issued % S::kSlots, use = issued / S::kSlots, i = issued / 2;
        if (issued == S::kSlots) wait_for_kernels_before();   // no slot is free again before
        if (use && !barrier_wait(empty + 8 * slot, (use - 1) & 1, &failed)) break;
        const bool by_masks = partial(i);
        load_rows<S>(ring_at + slot * S::kTile, issued & 1 ? &maps.dout : &maps.q, f.rows, chunk_of(i), token_of(i), kv_head, batch,
                     by_masks ? landed + 8 * (r % kRowRing) : full + 8 * slot);
        *static_cast<volatile uint32_t*>(&progress) = issued + 1;
        r += by_masks;
      }
      if (failed) {   // what is under way still lands before the CTA ends
        for (int i = 0; i < kWaitTries && !(barrier_try(k_full, 0) && barrier_try(v_full, 0)); i++) {}
        r = 0;
        for (int k = 0; k < issued; k++) {
          const bool by_masks = partial(k / 2);
          const uint32_t bar = by_masks ? landed + 8 * (r % kRowRing) : full + 8 * (k % S::kSlots), parity = (by_masks ? r / kRowRing : k / S::kSlots) & 1;
          r += by_masks;
          if (k < issued - S::kSlots) continue;
          for (int i = 0; i < kWaitTries && !barrier_try(bar, parity); i++) {}
        }
      }
    } else if (warp == 9 && n) {
      // -------------------------------------------------- products
      constexpr uint32_t kScores = product_descriptor<T>(128, 128, false), kResults = product_descriptor<T>(128, kDim, true);
      const int steps = (p.head_dim + 15) / 16;
      const uint32_t keys = low_half(at_address(tile_descriptor(16), k_at)), values = low_half(at_address(tile_descriptor(16), v_at)),
                     ring = low_half(at_address(tile_descriptor(16), ring_at)), ring_tokens = low_half(at_address(tile_descriptor(kBoxBytes), ring_at));
      const auto at_slot = [&](uint32_t slot) { return slot * (S::kTile >> 4); };
      const auto scores = [&](uint32_t slot) {
        product_of_tiles<kDim>(tmem, keys, ring + at_slot(slot), kScores, steps);
        products_done(s_full);
      };
      const auto dp = [&](uint32_t slot) {
        product_of_tiles<kDim>(tmem + dp_column, values, ring + at_slot(slot), kScores, steps);
        products_done(dp_full);
      };
      bool going = warp_wait3(k_full, 0, full, 0, 0, 0, &failed);
      if (going && elected()) scores(0);
      __syncwarp();
      going = going && warp_wait3(v_full, 0, full + 8, 0, 0, 0, &failed);
      if (going && elected()) dp(1);
      __syncwarp();
      wait_for_kernels_before();
      Ring<S::kSlots> q, g, next_q, next_g;   // queries and their gradients, of this tile and the next
      g.next();
      next_q.next(2);
      next_g.next(3);
#pragma unroll 1
      for (int i = 0; i < n && going; i++) {
        const bool more = i + 1 < n;
        going = warp_wait3(p_full, i & 1, more ? full + 8 * next_q.slot : 0, next_q.phase, 0, 0, &failed);
        if (!going) break;
        tmem_after_sync();
        if (elected()) {
          const uint32_t b = ring_tokens + at_slot(g.slot);
          product_over_tokens(tmem + dv_column, tmem, b, kResults, i > 0);
          product_over_tokens(tmem + dv_column, tmem + 64, b + kHalfTokens, kResults, true);
          if (more) scores(next_q.slot);   // overwrites P after it has been read
          products_done(empty + 8 * g.slot);
        }
        __syncwarp();
        going = warp_wait3(ds_full, i & 1, more ? full + 8 * next_g.slot : 0, next_g.phase, 0, 0, &failed);
        if (!going) break;
        tmem_after_sync();
        if (elected()) {
          const uint32_t b = ring_tokens + at_slot(q.slot);
          product_over_tokens(tmem + dk_column, tmem + dp_column, b, kResults, i > 0);
          product_over_tokens(tmem + dk_column, tmem + dp_column + 64, b + kHalfTokens, kResults, true);
          if (more) dp(next_g.slot);
          products_done(empty + 8 * q.slot);
          if (!more) products_done(done);
        }
        __syncwarp();
        q.next(2);
        g.next(2);
        next_q.next(2);
        next_g.next(2);
      }
      if (!going) products_end(ended);
    } else if (warp == 10) {
      // -------------------------------------------------- what is known of the rows; -infinity makes P = 0 where there is none
      wait_for_kernels_before();
      for (int i = 0; i < n; i++) {
        const int token = token_of(i), chunk = chunk_of(i);
        const float2* from = f.stats + ((static_cast<int64_t>(batch) * p.kv_heads + kv_head) * p.tokens + token) * p.group;
        float* to = reinterpret_cast<float*>(stats[i & 1]);
        float2 x[4];
        for (int k = 0; k < 4; k++) {
          const int row = k * 32 + lane, t = row / f.rows.heads, head = chunk * f.rows.heads + row % f.rows.heads;
          x[k] = row < tile_rows && token + t < length && head < p.group ? from[static_cast<int64_t>(t) * p.group + head] : make_float2(-INFINITY, 0.0f);
        }
        if (i >= 2 && !warp_wait(stats_empty + 8 * (i & 1), (i / 2 - 1) & 1, &failed)) break;
        for (int k = 0; k < 4; k++) {
          to[k * 32 + lane] = x[k].x;
          to[128 + k * 32 + lane] = x[k].y;
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(stats_full + 8 * (i & 1));
      }
    } else if (warp == 11) {
      // -------------------------------------------------- zeros in rows behind the sequence
      int r = 0;
      for (int item = 0; item < 2 * n; item++) {
        const int i = item / 2;
        if (!partial(i)) continue;
        if (item >= S::kSlots) wait_for_kernels_before();   // its copy begins behind that; those of items before do not
        if (!warp_wait_behind(landed + 8 * (r % kRowRing), r / kRowRing & 1, &failed, &progress)) break;
        const uint32_t at = ring_at + item % S::kSlots * S::kTile;
        for (int row = max(length - token_of(i), 0) * f.rows.heads + lane / 8; row < tile_rows; row += 4) {
          for (int x = 0; x < S::kBoxes; x++) store_zeros(at + x * kBoxBytes + row * 128 + (lane & 7) * 16);
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) barrier_arrive(full + 8 * (item % S::kSlots));
        r++;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------------------------------------------- a key belongs to two threads, one for each half of the rows of a tile
    const int half = warp / 4, row = threadIdx.x & 127, key = k0 + row;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const float c = p.scale * kLog2e;
    const bool there = key < length;
    const int tokens_end = key < p.sinks || p.window >= length ? length : min(length, key + p.window);   // of the queries that read the key
    const uint32_t mine = tmem + 64 * half + lanes;
    bool going = true;
    wait_for_kernels_before();
    for (int i = 0; i < n; i++) {
      uint32_t s[64];
      going = warp_wait(stats_full + 8 * (i & 1), i / 2 & 1, &failed) && warp_wait(s_full, i & 1, &failed);
      if (!going) break;
      tmem_after_sync();
      tmem_load<32>(mine, s);
      tmem_load<32>(mine + 32, s + 32);
      tmem_loaded(s);
      const float4* lse = stats[i & 1][0] + 16 * half;
      const float4* delta = stats[i & 1][1] + 16 * half;
      const int token = token_of(i), lo = min(max(key - token, 0), f.rows.tokens), hi = there ? min(max(tokens_end - token, 0), f.rows.tokens) : 0;
      // rows beyond a box are zeros with P = 0 by their stats, so a whole tile needs no bits
      const uint64_t read = bits_of(64 * half, lo * f.rows.heads, hi == f.rows.tokens ? 128 : hi * f.rows.heads);
      const bool every = __all_sync(~0u, read == ~uint64_t{0});
#pragma unroll
      for (int x = 0; x < 2; x++) {
        uint32_t packed[16];
        const uint32_t word = static_cast<uint32_t>(read >> (32 * x));
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 l = lse[8 * x + k / 4];
          uint32_t* e = s + 32 * x + k;
          const float2 a = fma2(make_float2(__uint_as_float(e[0]), __uint_as_float(e[1])), make_float2(c, c), make_float2(l.x, l.y));
          const float2 b = fma2(make_float2(__uint_as_float(e[2]), __uint_as_float(e[3])), make_float2(c, c), make_float2(l.z, l.w));
          const float v[4] = {exp2_of(a.x), exp2_of(a.y), exp2_of(b.x), exp2_of(b.y)};
#pragma unroll
          for (int y = 0; y < 4; y++) e[y] = __float_as_uint(v[y]);
          if (!every) {
#pragma unroll
            for (int y = 0; y < 4; y++) e[y] = word >> (k + y) & 1 ? e[y] : 0u;
          }
          packed[k / 2] = pack2<T>(__uint_as_float(e[0]), __uint_as_float(e[1]));
          packed[k / 2 + 1] = pack2<T>(__uint_as_float(e[2]), __uint_as_float(e[3]));
        }
        tmem_store<16>(mine + 16 * x, packed);
      }
      tmem_stored();
      tmem_before_sync();
      warp_arrive(p_full, lane);
      going = warp_wait(dp_full, i & 1, &failed);
      if (!going) break;
      tmem_after_sync();
#pragma unroll
      for (int x = 0; x < 2; x++) {
        uint32_t d[32], packed[16];
        const uint32_t word = static_cast<uint32_t>(read >> (32 * x));
        tmem_load<32>(mine + dp_column + 32 * x, d);
        tmem_loaded(d);
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 l = delta[8 * x + k / 4];
          const uint32_t* e = s + 32 * x + k;
          float2 a = mul2(add2(make_float2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), make_float2(-l.x, -l.y)),
                          make_float2(__uint_as_float(e[0]), __uint_as_float(e[1])));
          float2 b = mul2(add2(make_float2(__uint_as_float(d[k + 2]), __uint_as_float(d[k + 3])), make_float2(-l.z, -l.w)),
                          make_float2(__uint_as_float(e[2]), __uint_as_float(e[3])));
          if (!every) {   // not 0 times an infinity
            a.x = word >> k & 1 ? a.x : 0.0f;
            a.y = word >> (k + 1) & 1 ? a.y : 0.0f;
            b.x = word >> (k + 2) & 1 ? b.x : 0.0f;
            b.y = word >> (k + 3) & 1 ? b.y : 0.0f;
          }
          packed[k / 2] = pack2<T>(a.x, a.y);
          packed[k / 2 + 1] = pack2<T>(b.x, b.y);
        }
        tmem_store<16>(mine + dp_column + 16 * x, packed);
      }
      warp_arrive(stats_empty + 8 * (i & 1), lane);
      tmem_stored();
      tmem_before_sync();
      warp_arrive(ds_full, lane);
    }
    if (n && going) going = warp_wait(done, 0, &failed);
    if (going && split) {   // the first warpgroup writes dV, the second dK
      tmem_after_sync();
      float* to = f.partial + ((((static_cast<int64_t>(job.part) * p.batch + batch) * p.kv_heads + kv_head) * f.sink_tiles + job.tile) * 2 + (half ? 0 : 1)) * 128 * p.head_dim + row * p.head_dim;
#pragma unroll
      for (int x = 0; x < kDim; x += 32) {
        uint32_t o[32] = {};
        if (n) {
          tmem_load<32>(tmem + (half ? dk_column : dv_column) + lanes + x, o);
          tmem_loaded(o);
        }
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          if (x + k < p.head_dim) *reinterpret_cast<float4*>(to + x + k) = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
        }
      }
    } else if (going) {   // the first warpgroup writes dV, the second dK
      tmem_after_sync();
      const Heads& out = half ? p.dk : p.dv;
      T* const to = reinterpret_cast<T*>(out.data) + batch * out.batch + key * out.token + kv_head * out.head;
      // keys behind the sequence get zeros, whatever they are; their accumulators are zeros but for what is not a number
      write_row<T, kDim>(tmem + (half ? dk_column : dv_column) + lanes, to, 0, p.head_dim, half ? p.scale : 1.0f, key < p.tokens, there && n > 0, n == 0);
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 9) tmem_free<512>(tmem);
  if (failed) {
    const KeyJob at = key_job_of(f, block_again());
    const int from = at.tile * 128, end = min(from + 128, p.tokens);
    if (at.tile < f.sink_tiles && f.sink_parts > 1) {
      float* to = f.partial + (((static_cast<int64_t>(at.part) * p.batch + at.batch) * p.kv_heads + at.kv_head) * f.sink_tiles + at.tile) * 256 * p.head_dim;
      for (int i = threadIdx.x; i < 256 * p.head_dim; i += kKeyThreads) to[i] = NAN;
    } else {
      spoil_rows(p.dk, at.batch, at.kv_head, from, end, p.head_dim);
      spoil_rows(p.dv, at.batch, at.kv_head, from, end, p.head_dim);
    }
    if (threadIdx.x == 0) *p.status = 1;
  }
}

// The parts of first tokens' gradients, added in order: a CTA a tile, dk or dv, some of its rows.
constexpr int kSumRows = 16;

template <class T>
__global__ void __launch_bounds__(128) causal_sum_kernel(const __grid_constant__ BackwardParams f) {
  const CausalParams& p = f.p;
  int id = blockIdx.x;
  const int rows = id % (128 / kSumRows) * kSumRows;
  id /= 128 / kSumRows;
  const int which = id % 2;     // dk, dv
  id /= 2;
  const int tile = id % f.sink_tiles, of = id / f.sink_tiles, kv_head = of % p.kv_heads, batch = of / p.kv_heads;
  const int length = sequence_of<false>(p, batch).fresh;
  const Heads& out = which ? p.dv : p.dk;
  const float by = which ? 1.0f : p.scale;
  const int64_t step = static_cast<int64_t>(p.batch) * p.kv_heads * f.sink_tiles * 256 * p.head_dim;
  const float* from = f.partial + ((static_cast<int64_t>(of) * f.sink_tiles + tile) * 2 + which) * 128 * p.head_dim;
  wait_for_kernels_before();
  for (int i = threadIdx.x; i < kSumRows * p.head_dim / 4; i += 128) {
    const int row = rows + 4 * i / p.head_dim, e = 4 * i % p.head_dim, key = tile * 128 + row;
    if (key >= p.tokens) continue;
    float4 sum = {};
    if (key < length) {
      for (int part = 0; part < f.sink_parts; part++) {
        const float4 x = *reinterpret_cast<const float4*>(from + part * step + row * p.head_dim + e);
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
      }
    }
    T* to = reinterpret_cast<T*>(out.data) + batch * out.batch + key * out.token + kv_head * out.head + e;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(sum.x * by, sum.y * by), pack2<T>(sum.z * by, sum.w * by));
  }
}

BackwardParams backward_plan(const CausalParams& p) {
  BackwardParams f = {};
  f.p = p;
  f.rows = row_tiles(p);
  f.sink_parts = 1;
  if (p.sinks && p.window < p.tokens) {
    f.sink_tiles = (std::min(p.sinks, p.tokens) + 127) / 128;
    // Parts as long as the rows of other tiles, and not too short; no more than kSplitCtas CTAs in all, which fill the device several times
    // over, since each leaves a tile of float32 sums (134 MB for heads of 128).  Both passes of the backward, 32 heads on 8: 32768 tokens,
    // window 512, 16384 first ones 22.1 ms with one part (0.4 GB more than the tensors), 27.0 with 32 (4.7 GB); 16 x 8192 tokens, window
    // 128, 4 first ones 4.38 ms with 8 parts, 4.47 with 16.
    const int64_t others = (static_cast<int64_t>(p.window) + 127) / f.rows.tokens + 2, all = f.rows.tiles;
    const int64_t most = std::min<int64_t>(32, kSplitCtas / (static_cast<int64_t>(p.batch) * p.kv_heads * f.sink_tiles));
    f.sink_parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, all / std::max<int64_t>(others, 16))));
  }
  return f;
}

size_t stats_bytes(const CausalParams& p) { return (sizeof(float2) * p.batch * p.q_heads * p.tokens + 15) / 16 * 16; }

template <class T, int kDim>
cudaError_t launch(const BackwardParams& f, const CausalMaps& maps, cudaStream_t stream) {
  constexpr int bytes = Sizes<kDim>::kShared;
  const CausalParams& p = f.p;
  cudaError_t e = allow_shared<causal_dq_kernel<T, kDim>>(bytes, p.device);
  if (e == cudaSuccess) e = allow_shared<causal_dkv_kernel<T, kDim>>(bytes, p.device);
  if (e != cudaSuccess) return e;
  const int64_t heads = static_cast<int64_t>(p.kv_heads) * p.batch;
  e = launch_behind(causal_dq_kernel<T, kDim>, dim3(static_cast<unsigned>(heads * f.rows.tiles * f.rows.chunks)), kRowThreads, bytes, stream, 1, f, maps);
  if (e != cudaSuccess) return e;
  e = launch_behind(causal_dkv_kernel<T, kDim>, dim3(static_cast<unsigned>(heads * ((p.tokens + 127) / 128 + f.sink_tiles * (f.sink_parts - 1)))), kKeyThreads, bytes,
                    stream, 1, f, maps);
  if (e != cudaSuccess || f.sink_parts == 1) return e;
  return launch_behind(causal_sum_kernel<T>, dim3(static_cast<unsigned>(heads * f.sink_tiles * 2 * (128 / kSumRows))), 128, 0, stream, 1, f);
}

}  // namespace

size_t backward_workspace(const CausalParams& p) {
  const BackwardParams f = backward_plan(p);
  const size_t partial = f.sink_parts > 1 ? sizeof(float) * f.sink_parts * p.batch * p.kv_heads * f.sink_tiles * 256 * p.head_dim : 0;
  return stats_bytes(p) + partial;
}

cudaError_t launch_causal_backward(const CausalParams& p, void* workspace, const CausalMaps& maps, int dtype, cudaStream_t stream) {
  BackwardParams f = backward_plan(p);
  f.stats = static_cast<float2*>(workspace);
  f.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(p));
  if (dtype == MLXD_F16) return p.head_dim > 64 ? launch<__half, 128>(f, maps, stream) : launch<__half, 64>(f, maps, stream);
  return p.head_dim > 64 ? launch<__nv_bfloat16, 128>(f, maps, stream) : launch<__nv_bfloat16, 64>(f, maps, stream);
}

}  // namespace mlxd
