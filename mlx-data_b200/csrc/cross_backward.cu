// Gradients of cross attention: one kernel for queries, one for keys and values.  Each works out the scores again, so that
// every sum has one owner and the same order in every call: no atomics, no sums through memory.  That is seven products of
// 128 x 128 x D for the five of the definition.  P and dS are rounded to 16 bits, since the tensor cores take both operands of one 16-bit
// type: errors of 1.4 roundings instead of one, with delta's share 1.6 at most.  A small dS of float16 is not scaled up ahead of it,
// since the gradients may come in near the largest float16 by a loss scale, and a large one not held at 65504, so that a loss scaler sees
// an infinity.  Measured: 2 x 2048 tokens, 4096 keys, 32 heads on 8, D = 128: 897 us, 766 TFLOP/s by the five, 1073 by the seven; D = 64:
// 625 us.  With few queries (8 x 255 tokens, 1024 keys, 12 heads of 80, padded grids: 83 us) a CTA's beginning and end are most of it:
// six rounds of CTAs with two tiles of queries each.
#include "cross.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kThreads = 384;          // two warpgroups for what lies between the products, then warps for copies, products, helpers
constexpr int kMaskRing = 4;
constexpr float kLog2e = 1.4426950408889634f;

template <int kDim>
struct Sizes {
  static constexpr int kTile = 128 * kDim * 2;             // bytes of 128 tokens
  static constexpr int kBoxes = kDim / 64;
  static constexpr int kSlots = kDim == 128 ? 5 : 8;       // of the ring
  static constexpr int kShared = (2 + kSlots) * kTile;
};

template <class S>
__device__ __forceinline__ void load_tile(uint32_t to, const CUtensorMap* map, int token, int head, int batch, uint32_t bar) {
  barrier_expect(bar, S::kTile);
  for (int x = 0; x < S::kBoxes; x++) tile_load(to + x * kBoxBytes, map, 64 * x, token, head, batch, bar);
}

// The accumulators of a row, scaled, rounded and put where a store of the tile finds them; zeros where there are none.
template <class T, int kDim>
__device__ __forceinline__ void stage_row(uint32_t tmem, uint32_t to, int row, float by, bool none) {
#pragma unroll
  for (int x = 0; x < kDim; x += 32) {
    uint32_t o[32] = {};
    if (!none) {
      tmem_load<32>(tmem + x, o);
      tmem_loaded(o);
    }
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = pack2<T>(__uint_as_float(o[k + 2 * i]) * by, __uint_as_float(o[k + 2 * i + 1]) * by);
      const int unit = (x + k) % 64 / 8;
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                   : : "r"(to + (x + k) / 64 * kBoxBytes + row * 128 + ((unit ^ (row & 7)) * 16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
  }
}

template <class S>
__device__ __forceinline__ void store_tile(const CUtensorMap* map, int dim, int token, int head, int batch, uint32_t from) {
  for (int x = 0; x < S::kBoxes && 64 * x < dim; x++) tile_store(map, 64 * x, token, head, batch, from + x * kBoxBytes);
  tile_stores_read();
}

// Of a row and this thread's half of the one tile of keys that there is: sums of P dP and of P, over the keys that are read.  Scores and
// dP stay where they are.  Where a wait runs out the caller's next one does too.
__device__ __forceinline__ void row_sums(uint32_t at, uint32_t dp_column, uint32_t s_full, uint32_t dp_full, uint32_t masked, bool partial,
                                         const uint32_t (&mask)[4], int half, float c, float base, volatile int* failed, float* sum,
                                         float* weights) {
  if (partial && !warp_wait(masked, 0, failed)) return;
  const uint32_t words[2] = {partial ? mask[2 * half] : ~0u, partial ? mask[2 * half + 1] : ~0u};
  const bool single = partial && __popc(mask[0]) + __popc(mask[1]) + __popc(mask[2]) + __popc(mask[3]) == 1;
  if (!warp_wait(s_full, 0, failed) || !warp_wait(dp_full, 0, failed)) return;
  tmem_after_sync();
  float total = 0, part = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t s[16], d[16];
    tmem_load<16>(at + 16 * i, s);
    tmem_load<16>(at + dp_column + 16 * i, d);
    tmem_loaded(s);
    tmem_loaded(d);
#pragma unroll
    for (int k = 0; k < 16; k++) {
      if (words[i / 2] >> (16 * (i & 1) + k) & 1) {
        // lse of the forward pass makes the one weight 1 but for a rounding
        const float w = exp2_of(fmaf(__uint_as_float(s[k]), c, base)), exact = single && w > 0 ? 1.0f : w;
        total += exact;
        part = fmaf(exact, __uint_as_float(d[k]), part);
      }
    }
  }
  *sum = part;
  *weights = total;
}

// dQ = scale dS K for 128 queries: S = Q K^T, P = exp(S - lse), dP = dO V^T, dS = P (dP - delta).  lse has the derivative P by S, so its
// gradient is taken off delta.  Two sets of scores, so that the
// products of the next tile run beside the exponentials of this one.  Also works out delta = sum(dO O) - dlse of its rows, which the
// other kernel reads.  O comes in rounded to 16 bits, and where few keys have weights dS is the small difference of dP and delta: with
// two keys dQ and dK were off by 0.0052 of their size in bfloat16 (the rounding of results alone: 0.0017).  So where a sample's keys
// fit one tile, whose P and dP are there before any dS, delta = sum(P dP) / sum(P) of these.  A single key has the weight 1, so that its
// dS is 0 and no remainder of a rounding.
template <class T, int kDim>
__global__ void __launch_bounds__(kThreads, 1) cross_dq_kernel(const __grid_constant__ CrossParams p, const __grid_constant__ CrossMaps maps) {
  using S = Sizes<kDim>;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[2 + 2 * S::kSlots + 2 + 4 + 2 * kMaskRing + 1 + 1];
  __shared__ uint32_t mask_words[kMaskRing][4];
  __shared__ float delta_parts[2][2][128];   // of a row's two threads: sums, and with one tile of keys those of weights
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, reach;
  asm volatile("griddepcontrol.launch_dependents;");   // the other kernel's CTAs take the SMs that these leave
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t q_at = smem_address(shared), do_at = q_at + S::kTile, ring_at = do_at + S::kTile;
  const uint32_t q_full = smem_address(bars), do_full = q_full + 8, full = q_full + 16, empty = full + 8 * S::kSlots,
                 s_full = empty + 8 * S::kSlots, dp_full = s_full + 16, ds_full = dp_full + 8, done = ds_full + 8, delta_full = done + 8,
                 masked = delta_full + 8, landed = masked + 8 * kMaskRing, staged_full = landed + 8 * kMaskRing, ended = staged_full + 8;

  const int q_tiles = (p.q_tokens + 127) / 128;
  const int q0 = blockIdx.x % q_tiles * 128, head = blockIdx.x / q_tiles % p.q_heads, batch = blockIdx.x / q_tiles / p.q_heads;
  if (threadIdx.x == 0) {
    failed = reach = 0;
    for (const uint32_t bar : {q_full, do_full, s_full, s_full + 8, dp_full, done, ended}) barrier_init(bar, 1);
    for (const uint32_t bar : {ds_full, delta_full, staged_full}) barrier_init(bar, 8);
    for (int i = 0; i < S::kSlots; i++) {
      barrier_init(full + 8 * i, 1);
      barrier_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kMaskRing; i++) {
      barrier_init(masked + 8 * i, 1);
      barrier_init(landed + 8 * i, 1);
    }
    barrier_init_done();
  }
  if (warp == 9) tmem_alloc<512>(smem_address(&tmem_slot));
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tmem = tmem_slot, dp_column = 256, dq_column = 384;   // scores in 0 and 128
  const int length = reach_of(p, batch, length_of(p, batch), &reach), n = (length + 127) / 128;
  const auto partial = [&](int j) { return p.key_mask != nullptr || (j + 1) * 128 > length; };
  const auto ring_of = [&](int j) { return p.key_mask ? j : 0; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 8 && lane == 0 && n) {
      // -------------------------------------------------- copies: keys of tile 0, values of tile 0, keys of tile 1, ...
      load_tile<S>(q_at, &maps.q, q0, head, batch, q_full);
      load_tile<S>(do_at, &maps.dout, q0, head, batch, do_full);
      int issued = 0;
      for (; issued < 2 * n; issued++) {
        const int slot = issued % S::kSlots, use = issued / S::kSlots, j = issued / 2;
        if (use && !barrier_wait(empty + 8 * slot, (use - 1) & 1, &failed)) break;
        // keys of a tile that is not read as a whole go by way of the mask warp
        const uint32_t bar = !(issued & 1) && partial(j) ? landed + 8 * (ring_of(j) % kMaskRing) : full + 8 * slot;
        load_tile<S>(ring_at + slot * S::kTile, issued & 1 ? &maps.v : &maps.k, j * 128, head / p.group, batch, bar);
      }
      if (failed) {   // what is under way still lands before the CTA ends
        for (int i = 0; i < kWaitTries && !(barrier_try(q_full, 0) && barrier_try(do_full, 0)); i++) {}
        for (int k = max(0, issued - S::kSlots); k < issued; k++) {
          const int r = ring_of(k / 2);
          const bool masks = !(k & 1) && partial(k / 2);
          const uint32_t bar = masks ? landed + 8 * (r % kMaskRing) : full + 8 * (k % S::kSlots);
          for (int i = 0; i < kWaitTries && !barrier_try(bar, (masks ? r / kMaskRing : k / S::kSlots) & 1); i++) {}
        }
      }
    } else if (warp == 9 && n) {
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
      // one look at barriers between two groups of products: the tensor cores are not far behind the thread that issues them
      Ring<S::kSlots> k, v, next_k;          // keys of this tile, values of the next, keys of the one after
      v.next(3);
      next_k.next(4);
#pragma unroll 1
      for (int j = 0; j < n && going; j++) {
        going = warp_wait3(ds_full, j & 1, j + 1 < n ? full + 8 * v.slot : 0, v.phase, j + 2 < n ? full + 8 * next_k.slot : 0, next_k.phase, &failed);
        if (!going) break;
        tmem_after_sync();
        if (elected()) {
          if (j + 1 < n) dp(v.slot);
          const uint32_t ds = tmem + 128 * (j & 1), b = ring_tokens + at_slot(k.slot);
          product_over_tokens(tmem + dq_column, ds, b, kResults, j > 0);
          product_over_tokens(tmem + dq_column, ds + 64, b + kHalfTokens, kResults, true);
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
    } else if (warp == 10) {
      // -------------------------------------------------- masks: which keys are read, and zeros where they are not
      for (int j = 0; j < n; j++) {
        if (!partial(j)) continue;
        uint32_t words[4];
        for (int i = 0; i < 4; i++) {
          const int key = j * 128 + i * 32 + lane;
          words[i] = __ballot_sync(~0u, key < length && (!p.key_mask || p.key_mask[batch * p.key_mask_stride + key]));
        }
        const int item = 2 * j, r = ring_of(j);
        if (!warp_wait(landed + 8 * (r % kMaskRing), r / kMaskRing & 1, &failed)) break;
        const uint32_t keys = ring_at + item % S::kSlots * S::kTile;
        for (int i = 0; i < 4; i++) {
          if (lane == 0) mask_words[r % kMaskRing][i] = words[i];
          for (int row = lane / 8; row < 32; row += 4) {   // 8 lanes a row of 128 bytes
            if (words[i] >> row & 1) continue;
            for (int x = 0; x < S::kBoxes; x++) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                           : : "r"(keys + x * kBoxBytes + (32 * i + row) * 128 + (lane & 7) * 16), "r"(0) : "memory");
            }
          }
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) {
          barrier_arrive(full + 8 * (item % S::kSlots));
          barrier_arrive(masked + 8 * (r % kMaskRing));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------------------------------------------- a row belongs to two threads, one for each half of the keys of a tile
    const int half = warp / 4, row = threadIdx.x & 127;
    const bool there = q0 + row < p.q_tokens;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const int64_t stat = (static_cast<int64_t>(batch) * p.q_heads + head) * p.q_tokens + q0 + row;
    const float c = p.scale * kLog2e;
    // a row that is not there gets P = 0
    const float base = there ? row_base(p.lse[stat]) : -INFINITY;
    float part = 0, weights = 1;
    if (n == 1) {
      row_sums(tmem + 64 * half + lanes, dp_column, s_full, dp_full, masked, partial(0), mask_words[0], half, c, base, &failed, &part, &weights);
    } else if (there) {   // delta: this thread's half of the elements
      const T* o = reinterpret_cast<const T*>(p.out.data) + batch * p.out.batch + (q0 + row) * p.out.token + head * p.out.head;
      const T* g = reinterpret_cast<const T*>(p.dout.data) + batch * p.dout.batch + (q0 + row) * p.dout.token + head * p.dout.head;
#pragma unroll
      for (int x = 0; x < kDim / 2; x += 8) {
        const int at = half * (kDim / 2) + x;
        if (at < p.head_dim) {
          const uint4 a = *reinterpret_cast<const uint4*>(o + at), b = *reinterpret_cast<const uint4*>(g + at);
          const T *u = reinterpret_cast<const T*>(&a), *v = reinterpret_cast<const T*>(&b);
#pragma unroll
          for (int i = 0; i < 8; i++) part += static_cast<float>(u[i]) * static_cast<float>(v[i]);
        }
      }
    }
    delta_parts[0][half][row] = part;
    delta_parts[1][half][row] = weights;
    warp_arrive(delta_full, lane);
    bool going = warp_wait(delta_full, 0, &failed);
    float delta = going ? delta_parts[0][0][row] + delta_parts[0][1][row] : 0.0f;
    if (n == 1 && going) {
      weights = delta_parts[1][0][row] + delta_parts[1][1][row];
      delta = weights == 0 ? 0.0f : delta / weights;
    }
    if (p.lse_grad && there) delta -= p.lse_grad[stat];
    if (there && half == 0) p.delta[stat] = delta;
    for (int j = 0; j < n && going; j++) {
      const uint32_t mine = tmem + 128 * (j & 1) + 64 * half + lanes;
      uint32_t s[64];
      going = warp_wait(s_full + 8 * (j & 1), j / 2 & 1, &failed);
      if (!going) break;
      tmem_after_sync();
      tmem_load<32>(mine, s);
      tmem_load<32>(mine + 32, s + 32);
      tmem_loaded(s);
#pragma unroll
      for (int k = 0; k < 64; k += 2) {
        const float2 x = fma2(make_float2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), make_float2(c, c), make_float2(base, base));
        s[k] = __float_as_uint(exp2_of(x.x));
        s[k + 1] = __float_as_uint(exp2_of(x.y));
      }
      uint32_t words[2] = {~0u, ~0u};
      if (partial(j)) {
        const int r = ring_of(j);
        going = warp_wait(masked + 8 * (r % kMaskRing), r / kMaskRing & 1, &failed);
        if (!going) break;
        words[0] = mask_words[r % kMaskRing][2 * half];
        words[1] = mask_words[r % kMaskRing][2 * half + 1];
      }
      going = warp_wait(dp_full, j & 1, &failed);
      if (!going) break;
      tmem_after_sync();
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t d[32], packed[16];
        tmem_load<32>(tmem + dp_column + 64 * half + 32 * i + lanes, d);
        tmem_loaded(d);
        if (words[i] == ~0u) {
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 x = add2(make_float2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), make_float2(-delta, -delta));
            const float2 y = mul2(x, make_float2(__uint_as_float(s[32 * i + k]), __uint_as_float(s[32 * i + k + 1])));
            packed[k / 2] = pack2<T>(y.x, y.y);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float x = words[i] >> k & 1 ? (__uint_as_float(d[k]) - delta) * __uint_as_float(s[32 * i + k]) : 0.0f;
            const float y = words[i] >> (k + 1) & 1 ? (__uint_as_float(d[k + 1]) - delta) * __uint_as_float(s[32 * i + k + 1]) : 0.0f;
            packed[k / 2] = pack2<T>(x, y);
          }
        }
        tmem_store<16>(mine + 16 * i, packed);
      }
      tmem_stored();
      tmem_before_sync();
      warp_arrive(ds_full, lane);
    }
    if (n && going) going = warp_wait(done, 0, &failed);
    if (going) {
      tmem_after_sync();
      if (half == 0) stage_row<T, kDim>(tmem + dq_column + lanes, q_at, row, p.scale, n == 0);
      fence_async_proxy();
      warp_arrive(staged_full, lane);
      if (threadIdx.x == 0 && barrier_wait(staged_full, 0, &failed)) store_tile<S>(&maps.dq, p.head_dim, q0, head, batch, q_at);
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 9) tmem_free<512>(tmem);
  if (failed) {
    const int id = block_again(), tiles = (p.q_tokens + 127) / 128, from = id % tiles * 128, of = id / tiles;
    const int end = min(from + 128, p.q_tokens), i = from + static_cast<int>(threadIdx.x);
    spoil_rows(p.dq, of / p.q_heads, of % p.q_heads, from, end, p.head_dim);
    // the other kernel's results are not valid either
    if (i < end) p.delta[static_cast<int64_t>(of) * p.q_tokens + i] = NAN;
    if (threadIdx.x == 0) *p.status = 1;
  }
}

// dV = P^T dO and dK = scale dS^T Q for 128 keys, over the queries of every head that shares them.  Scores lie the other way round
// (a key a lane), so that P^T and dS^T are operands as they are.
template <class T, int kDim>
__global__ void __launch_bounds__(kThreads, 1) cross_dkv_kernel(const __grid_constant__ CrossParams p, const __grid_constant__ CrossMaps maps) {
  using S = Sizes<kDim>;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[2 + 2 * S::kSlots + 5 + 4 + 1 + 1];
  __shared__ float4 stats[2][2][32];      // of the queries of a tile: -lse * log2(e), delta
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, reach;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t k_at = smem_address(shared), v_at = k_at + S::kTile, ring_at = v_at + S::kTile;
  const uint32_t k_full = smem_address(bars), v_full = k_full + 8, full = k_full + 16, empty = full + 8 * S::kSlots,
                 s_full = empty + 8 * S::kSlots, dp_full = s_full + 8, p_full = dp_full + 8, ds_full = p_full + 8, done = ds_full + 8,
                 stats_full = done + 8, stats_empty = stats_full + 16, staged_full = stats_empty + 16, ended = staged_full + 8;

  const int k_tiles = (p.kv_tokens + 127) / 128;
  const int k0 = blockIdx.x % k_tiles * 128, kv_head = blockIdx.x / k_tiles % p.kv_heads, batch = blockIdx.x / k_tiles / p.kv_heads;
  const int q_tiles = (p.q_tokens + 127) / 128;

  if (threadIdx.x == 0) {
    failed = reach = 0;
    for (const uint32_t bar : {k_full, v_full, s_full, dp_full, done, stats_full, stats_full + 8, ended}) barrier_init(bar, 1);
    for (const uint32_t bar : {p_full, ds_full, staged_full}) barrier_init(bar, 8);
    for (const uint32_t bar : {stats_empty, stats_empty + 8}) barrier_init(bar, 8);
    for (int i = 0; i < S::kSlots; i++) {
      barrier_init(full + 8 * i, 1);
      barrier_init(empty + 8 * i, 1);
    }
    barrier_init_done();
  }
  if (warp == 9) tmem_alloc<512>(smem_address(&tmem_slot));
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tmem = tmem_slot, dp_column = 128, dv_column = 256, dk_column = 384;   // scores in 0
  const int length = reach_of(p, batch, length_of(p, batch), &reach);
  const int n = k0 < length ? q_tiles * p.group : 0;   // tiles of queries, head by head

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 8 && lane == 0 && n) {
      // -------------------------------------------------- copies: queries of tile 0, their gradients, queries of tile 1, ...
      load_tile<S>(k_at, &maps.k, k0, kv_head, batch, k_full);
      load_tile<S>(v_at, &maps.v, k0, kv_head, batch, v_full);
      int issued = 0;
      for (; issued < 2 * n; issued++) {
        const int slot = issued % S::kSlots, use = issued / S::kSlots, i = issued / 2;
        if (issued == S::kSlots) wait_for_kernels_before();   // no slot is free again before
        if (use && !barrier_wait(empty + 8 * slot, (use - 1) & 1, &failed)) break;
        load_tile<S>(ring_at + slot * S::kTile, issued & 1 ? &maps.dout : &maps.q, i % q_tiles * 128, kv_head * p.group + i / q_tiles, batch, full + 8 * slot);
      }
      if (failed) {   // what is under way still lands before the CTA ends
        for (int i = 0; i < kWaitTries && !(barrier_try(k_full, 0) && barrier_try(v_full, 0)); i++) {}
        for (int k = max(0, issued - S::kSlots); k < issued; k++) {
          for (int i = 0; i < kWaitTries && !barrier_try(full + 8 * (k % S::kSlots), k / S::kSlots & 1); i++) {}
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
      // -------------------------------------------------- what is known of the queries; -infinity makes P = 0 where there is none
      wait_for_kernels_before();   // delta comes from there
      for (int i = 0; i < n; i++) {
        const int64_t first = (static_cast<int64_t>(batch) * p.q_heads + kv_head * p.group + i / q_tiles) * p.q_tokens;
        float* to = reinterpret_cast<float*>(stats[i & 1]);
        float lse[4], delta[4];
        for (int k = 0; k < 4; k++) {
          const int token = i % q_tiles * 128 + k * 32 + lane;
          lse[k] = token < p.q_tokens ? row_base(p.lse[first + token]) : -INFINITY;
          delta[k] = token < p.q_tokens ? p.delta[first + token] : 0.0f;
        }
        if (i >= 2 && !warp_wait(stats_empty + 8 * (i & 1), (i / 2 - 1) & 1, &failed)) break;
        for (int k = 0; k < 4; k++) {
          to[k * 32 + lane] = lse[k];
          to[128 + k * 32 + lane] = delta[k];
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(stats_full + 8 * (i & 1));
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------------------------------------------- a key belongs to two threads, one for each half of the queries of a tile
    const int half = warp / 4, row = threadIdx.x & 127, key = k0 + row;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const float c = p.scale * kLog2e;
    const bool read = key < length && (!p.key_mask || p.key_mask[batch * p.key_mask_stride + key]);
    const uint32_t mine = tmem + 64 * half + lanes;
    const int end = p.q_tokens - 128 * (q_tiles - 1) - 64 * half;   // of this thread's queries in the last tile of a head
    int ragged = end < 64 ? q_tiles - 1 : -1;                       // the next such tile that has not all of them
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
      // queries that are not there are zeros, whose scores are not a number where a key holds an infinity
      if (i == ragged) {
        ragged += q_tiles;
#pragma unroll
        for (int k = 0; k < 64; k++) {
          if (k >= end) s[k] = 0;
        }
      }
      const float4* lse = stats[i & 1][0] + 16 * half;
      const float4* delta = stats[i & 1][1] + 16 * half;
#pragma unroll
      for (int x = 0; x < 2; x++) {
        uint32_t packed[16];
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 l = lse[8 * x + k / 4];
          uint32_t* e = s + 32 * x + k;
          const float2 a = fma2(make_float2(__uint_as_float(e[0]), __uint_as_float(e[1])), make_float2(c, c), make_float2(l.x, l.y));
          const float2 b = fma2(make_float2(__uint_as_float(e[2]), __uint_as_float(e[3])), make_float2(c, c), make_float2(l.z, l.w));
          const float v[4] = {exp2_of(a.x), exp2_of(a.y), exp2_of(b.x), exp2_of(b.y)};
#pragma unroll
          for (int y = 0; y < 4; y++) e[y] = read ? __float_as_uint(v[y]) : 0u;
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
        tmem_load<32>(mine + dp_column + 32 * x, d);
        tmem_loaded(d);
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 l = delta[8 * x + k / 4];
          const uint32_t* e = s + 32 * x + k;
          const float2 a = mul2(add2(make_float2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), make_float2(-l.x, -l.y)),
                                make_float2(__uint_as_float(e[0]), __uint_as_float(e[1])));
          const float2 b = mul2(add2(make_float2(__uint_as_float(d[k + 2]), __uint_as_float(d[k + 3])), make_float2(-l.z, -l.w)),
                                make_float2(__uint_as_float(e[2]), __uint_as_float(e[3])));
          packed[k / 2] = read ? pack2<T>(a.x, a.y) : 0u;
          packed[k / 2 + 1] = read ? pack2<T>(b.x, b.y) : 0u;
        }
        tmem_store<16>(mine + dp_column + 16 * x, packed);
      }
      warp_arrive(stats_empty + 8 * (i & 1), lane);
      tmem_stored();
      tmem_before_sync();
      warp_arrive(ds_full, lane);
    }
    if (n && going) going = warp_wait(done, 0, &failed);
    // keys that are not read get zeros, not 0 times an infinity in queries or in the result's gradient
    if (going) {   // the first warpgroup stores dV, the second dK, out of the ring, which is no longer needed
      tmem_after_sync();
      const uint32_t staged = ring_at + half * S::kTile;
      stage_row<T, kDim>(tmem + (half ? dk_column : dv_column) + lanes, staged, row, half ? p.scale : 1.0f, n == 0);
      if (n && !read) {
#pragma unroll
        for (int unit = 0; unit < kDim / 8; unit++) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                       : : "r"(staged + unit / 8 * kBoxBytes + row * 128 + ((unit % 8 ^ (row & 7)) * 16)), "r"(0) : "memory");
        }
      }
      fence_async_proxy();
      warp_arrive(staged_full, lane);
      if (row == 0 && barrier_wait(staged_full, 0, &failed)) store_tile<S>(half ? &maps.dk : &maps.dv, p.head_dim, k0, kv_head, batch, staged);
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 9) tmem_free<512>(tmem);
  if (failed) {
    const int id = block_again(), tiles = (p.kv_tokens + 127) / 128, from = id % tiles * 128, of = id / tiles;
    const int end = min(from + 128, p.kv_tokens);
    spoil_rows(p.dk, of / p.kv_heads, of % p.kv_heads, from, end, p.head_dim);
    spoil_rows(p.dv, of / p.kv_heads, of % p.kv_heads, from, end, p.head_dim);
    if (threadIdx.x == 0) *p.status = 1;
  }
}

template <class T, int kDim>
cudaError_t launch(const CrossParams& p, const CrossMaps& maps, cudaStream_t stream) {
  constexpr int bytes = Sizes<kDim>::kShared;
  if (p.q_tokens) {
    const cudaError_t e = allow_shared<cross_dq_kernel<T, kDim>>(bytes, p.device);
    if (e != cudaSuccess) return e;
    cross_dq_kernel<T, kDim><<<static_cast<unsigned>((p.q_tokens + 127) / 128) * p.q_heads * p.batch, kThreads, bytes, stream>>>(p, maps);
  }
  if (p.kv_tokens) {
    const cudaError_t e = allow_shared<cross_dkv_kernel<T, kDim>>(bytes, p.device);
    if (e != cudaSuccess) return e;
    // begins while the last CTAs of the kernel before run; what it needs of that one it waits for on the device
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>((p.kv_tokens + 127) / 128) * p.kv_heads * p.batch);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = p.q_tokens ? 1 : 0;
    const cudaError_t launched = cudaLaunchKernelEx(&config, cross_dkv_kernel<T, kDim>, p, maps);
    if (launched != cudaSuccess) return launched;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cross_backward(const CrossParams& p, const CrossMaps& maps, int dtype, cudaStream_t stream) {
  if (dtype == MLXD_F16) return p.head_dim > 64 ? launch<__half, 128>(p, maps, stream) : launch<__half, 64>(p, maps, stream);
  return p.head_dim > 64 ? launch<__nv_bfloat16, 128>(p, maps, stream) : launch<__nv_bfloat16, 64>(p, maps, stream);
}

}  // namespace mlxd
