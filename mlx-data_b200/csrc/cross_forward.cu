// Cross attention of many queries: two tiles of 128 query rows a CTA against tiles of 128 keys.
//
// One pass over the keys with a running maximum m and sum l of each row: S = Q K^T, P = 2^(c S - c m) with c = scale log2(e), O = O + P V,
// O and l scaled where m moves; at last O / l.  4 Sq Sk D operations, so the tensor cores are the floor; the exponentials (one
// for 4 D operations) take as long at D = 128 and twice as long at 64.  Scores and results stay in tensor memory (512 columns: two tiles of
// 128 scores and 128 results each), weights go back where their scores were and are an operand from there.  While one tile of rows is in
// the tensor cores the other is with the softmax.  A row belongs to two threads, so that a tile's softmax takes half as long: it and the
// products of a tile follow one another (about 1600 and 1300 cycles, of which 1024 are products), and a tile waits for both.
// Measured: 2 x 2048 tokens, 6404 keys, 32 heads on 8, D = 128: 393 us, 1094 TFLOP/s (67 % of the measured rate; 440 us where calls
// follow one another for long and the power cap lowers the clock); D = 64, 4096 keys: 222 us, 619.
#include "cross.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kThreads = 640;          // four warpgroups of softmax, then warps for copies, products, masks
constexpr int kMaskRing = 4;
constexpr float kLog2e = 1.4426950408889634f;
// A row's reference maximum is moved, and what is summed so far scaled, only where its weight has grown by more than
// 2^8: the result is the same quotient, and 2^8 is far from the largest float16.
constexpr float kSlack = 8.0f;
// Of eight pairs of exponentials so many are worked out by multiply-adds: the pipe of exponentials is what a tile of scores waits
// for.  Measured for 0, 1, 2, 3: 398, 393, 392, 400 us (2 x 2048 tokens, 6404 keys, 32 heads of 128), 224, 222, 225, 232 us (4096
// keys, heads of 64): above one or two in eight the issue of instructions takes as long.
constexpr int kByFma = 1;

template <int kDim>
struct Sizes {
  static constexpr int kTile = 128 * kDim * 2;             // bytes of 128 tokens
  static constexpr int kBoxes = kDim / 64;
  static constexpr int kSlots = kDim == 128 ? 5 : 8;       // of the ring of keys and values
  static constexpr int kShared = (2 + kSlots) * kTile;
};

// 64 scores of a row.
__device__ __forceinline__ void load_scores(uint32_t at, uint32_t (&s)[64]) {
  tmem_load<32>(at, s);
  tmem_load<32>(at + 32, s + 32);
  tmem_loaded(s);
}

// -infinity where a key is not read.
__device__ __forceinline__ void mask_scores(uint32_t word0, uint32_t word1, uint32_t (&s)[64]) {
#pragma unroll
  for (int k = 0; k < 32; k++) {
    if (!(word0 >> k & 1)) s[k] = __float_as_uint(-INFINITY);
    if (!(word1 >> k & 1)) s[32 + k] = __float_as_uint(-INFINITY);
  }
}

__device__ __forceinline__ float most_of(const uint32_t (&s)[64]) {
  float most[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    most[i] = __uint_as_float(s[i]);
#pragma unroll
    for (int k = 1; k < 16; k++) most[i] = fmaxf(most[i], __uint_as_float(s[i + 4 * k]));
  }
  return fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
}

// exp(score - maximum) of 64 scores, as 2^(c s + base): summed in float32, rounded to 16 bits (the tensor cores take both operands of one
// 16-bit type; the result's error becomes 1.4 roundings instead of one), stored in the first 32 columns of where they came from.
template <class T>
__device__ __forceinline__ void weigh(const uint32_t (&s)[64], float c, float base, float2 (&sum)[2], uint32_t to) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    uint32_t packed[16];
#pragma unroll
    for (int k = 0; k < 16; k++) {
      float2 x = make_float2(__uint_as_float(s[32 * i + 2 * k]), __uint_as_float(s[32 * i + 2 * k + 1]));
      x = fma2(x, make_float2(c, c), make_float2(base, base));
      if (k % 8 < kByFma) {
        x = exp2_by_fma(x);
      } else {
        x.x = exp2_of(x.x);
        x.y = exp2_of(x.y);
      }
      sum[k & 1] = add2(sum[k & 1], x);
      packed[k] = pack2<T>(x.x, x.y);
    }
    tmem_store<16>(to + 16 * i, packed);
  }
}

template <class T, int kDim>
__global__ void __launch_bounds__(kThreads, 1) cross_forward_kernel(const __grid_constant__ CrossParams p, const __grid_constant__ CrossMaps maps) {
  using S = Sizes<kDim>;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[2 + 2 * S::kSlots + 6 + 2 * kMaskRing + 2 + 1];
  __shared__ uint32_t mask_words[kMaskRing][4];
  __shared__ float exchange[2][2][128];   // of a row's two threads: maxima, sums at last
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, reach;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t tiles_at = smem_address(shared), ring_at = tiles_at + 2 * S::kTile;
  const uint32_t q_full = smem_address(bars), full = q_full + 16, empty = full + 8 * S::kSlots, s_full = empty + 8 * S::kSlots,
                 p_full = s_full + 16, o_full = p_full + 16, masked = o_full + 16, landed = masked + 8 * kMaskRing, staged_full = landed + 8 * kMaskRing, ended = staged_full + 16;

  // CTAs of 256 rows first, head by head; those of a ragged end of at most 128 rows, which take less time, after all others, where
  // they fill the SMs that become free (333 rows, 96 heads: 31.9 us in order of tiles, 29.4 so).
  const int q_tiles = (p.q_tokens + 255) / 256, end_rows = p.q_tokens - 256 * (q_tiles - 1), whole = end_rows > 128 ? q_tiles : q_tiles - 1;
  const int wholes = whole * p.q_heads * p.batch;
  const auto rows_of = [&](int id) {
    const int of = id < wholes ? id / whole : id - wholes;
    return make_int3((id < wholes ? id % whole : q_tiles - 1) * 256, of % p.q_heads, of / p.q_heads);
  };
  const int3 mine_are = rows_of(blockIdx.x);
  const int q0 = mine_are.x, head = mine_are.y, batch = mine_are.z;
  const int rows = p.q_tokens - q0 > 128 ? 2 : 1;   // tiles of query rows
  if (threadIdx.x == 0) {
    failed = reach = 0;
    barrier_init(ended, 1);
    for (int t = 0; t < 2; t++) {
      barrier_init(q_full + 8 * t, 1);
      barrier_init(s_full + 8 * t, 1);
      barrier_init(p_full + 8 * t, 8);
      barrier_init(o_full + 8 * t, 1);
      barrier_init(staged_full + 8 * t, 8);
    }
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
  if (warp == 17) tmem_alloc<512>(smem_address(&tmem_slot));
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tmem = tmem_slot;
  const int length = reach_of(p, batch, length_of(p, batch), &reach), n = (length + 127) / 128;
  // tiles of keys of which some may not be read: every one under a mask, else the last
  const auto partial = [&](int j) { return p.key_mask != nullptr || (j + 1) * 128 > length; };
  const auto ring_of = [&](int j) { return p.key_mask ? j : 0; };
  const uint32_t o_column = 256;   // scores of tile t in columns 128 t, results in 256 + 128 t

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 16 && lane == 0 && n) {
      // -------------------------------------------------- copies
      for (int t = 0; t < rows; t++) {
        barrier_expect(q_full + 8 * t, S::kTile);
        for (int x = 0; x < S::kBoxes; x++) {
          tile_load(tiles_at + t * S::kTile + x * kBoxBytes, &maps.q, 64 * x, q0 + 128 * t, head, batch, q_full + 8 * t);
        }
      }
      int issued = 0;
      for (; issued < 2 * n; issued++) {   // keys of tile 0, values of tile 0, keys of tile 1, ...
        const int slot = issued % S::kSlots, use = issued / S::kSlots, j = issued / 2;
        if (use && !barrier_wait(empty + 8 * slot, (use - 1) & 1, &failed)) break;
        // values of a tile that is not read as a whole go by way of the mask warp
        const uint32_t bar = issued & 1 && partial(j) ? landed + 8 * (ring_of(j) % kMaskRing) : full + 8 * slot;
        barrier_expect(bar, S::kTile);
        for (int x = 0; x < S::kBoxes; x++) {
          tile_load(ring_at + slot * S::kTile + x * kBoxBytes, issued & 1 ? &maps.v : &maps.k, 64 * x, j * 128,
                    head / p.group, batch, bar);
        }
      }
      if (failed) {   // what is under way still lands before the CTA ends
        for (int t = 0; t < rows; t++) {
          for (int i = 0; i < kWaitTries && !barrier_try(q_full + 8 * t, 0); i++) {}
        }
        for (int k = max(0, issued - S::kSlots); k < issued; k++) {
          const int r = ring_of(k / 2);
          const bool masks = k & 1 && partial(k / 2);
          const uint32_t bar = masks ? landed + 8 * (r % kMaskRing) : full + 8 * (k % S::kSlots);
          for (int i = 0; i < kWaitTries && !barrier_try(bar, (masks ? r / kMaskRing : k / S::kSlots) & 1); i++) {}
        }
      }
    } else if (warp == 17 && n) {
      // -------------------------------------------------- products
      constexpr uint32_t kScores = product_descriptor<T>(128, 128, false), kResults = product_descriptor<T>(128, kDim, true);
      const int steps = (p.head_dim + 15) / 16;
      const uint32_t queries = low_half(at_address(tile_descriptor(16), tiles_at)), keys = low_half(at_address(tile_descriptor(16), ring_at)),
                     values = low_half(at_address(tile_descriptor(kBoxBytes), ring_at));
      const auto scores = [&](int t, uint32_t slot) {   // S = Q K^T
        product_of_tiles<kDim>(tmem + 128 * t, queries + t * (S::kTile >> 4), keys + slot * (S::kTile >> 4), kScores, steps);
        products_done(s_full + 8 * t);
      };
      Ring<S::kSlots> at;                               // the item that is needed next
      bool going = warp_wait(full, 0, &failed);
      for (int t = 0; t < rows && going; t++) {
        going = warp_wait(q_full + 8 * t, 0, &failed);
        if (going && elected()) {
          scores(t, 0);
          if (t + 1 == rows) products_done(empty + 0);
        }
        __syncwarp();
      }
      at.next();
      // The tensor cores run a product or two behind the thread that issues them, so between two groups of products there is one
      // look at barriers and no more: with the last group of a tile of keys, at those of the next one's tiles too.
      Ring<S::kSlots> v = at, k = at;
      k.next();
      going = going && warp_wait3(full + 8 * v.slot, v.phase, n > 1 ? full + 8 * k.slot : 0, k.phase, 0, 0, &failed);
#pragma unroll 1
      for (int j = 0; j < n && going; j++) {
        Ring<S::kSlots> next_v = k, next_k;
        next_v.next();
        next_k = next_v;
        next_k.next();
#pragma unroll 1
        for (int t = 0; t < rows && going; t++) {
          // O += P V, P where the scores were, when both halves of the keys have been weighed
          const uint32_t o = tmem + o_column + 128 * t, values_at = values + v.slot * (S::kTile >> 4);
          const bool last = t + 1 == rows;
          going = warp_wait3(p_full + 8 * t, j & 1, last && j + 1 < n ? full + 8 * next_v.slot : 0, next_v.phase,
                             last && j + 2 < n ? full + 8 * next_k.slot : 0, next_k.phase, &failed);
          if (!going) break;
          tmem_after_sync();
          if (elected()) {
            product_over_tokens(o, tmem + 128 * t, values_at, kResults, j > 0);
            product_over_tokens(o, tmem + 128 * t + 64, values_at + kHalfTokens, kResults, true);
            if (last) products_done(empty + 8 * v.slot);
            // products run in the order in which they are issued: these scores overwrite P after it has been read
            if (j + 1 < n) {
              scores(t, k.slot);
              if (last) products_done(empty + 8 * k.slot);
            } else {
              products_done(o_full + 8 * t);
            }
          }
          __syncwarp();
        }
        v = next_v;
        k = next_k;
      }
      if (!going) products_end(ended);
    } else if (warp == 19) {
      // -------------------------------------------------- masks: which keys are read, and zeros where values are not
      for (int j = 0; j < n; j++) {
        if (!partial(j)) continue;
        uint32_t words[4];
        for (int i = 0; i < 4; i++) {
          const int key = j * 128 + i * 32 + lane;
          words[i] = __ballot_sync(~0u, key < length && (!p.key_mask || p.key_mask[batch * p.key_mask_stride + key]));
        }
        const int item = 2 * j + 1, r = ring_of(j);
        if (!warp_wait(landed + 8 * (r % kMaskRing), r / kMaskRing & 1, &failed)) break;
        const uint32_t values = ring_at + item % S::kSlots * S::kTile;
        for (int i = 0; i < 4; i++) {
          if (lane == 0) mask_words[r % kMaskRing][i] = words[i];
          // 8 lanes a row of 128 bytes
          for (int row = lane / 8; row < 32; row += 4) {
            if (words[i] >> row & 1) continue;
            for (int x = 0; x < S::kBoxes; x++) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                           : : "r"(values + x * kBoxBytes + (32 * i + row) * 128 + (lane & 7) * 16), "r"(0) : "memory");
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------------------------------------------- softmax: a row belongs to two threads, one for each half of the keys of a tile
    // A wait that ran out does not end the loop: the two warps of a row's threads meet at a barrier for every tile.
    const int t = warp / 8, half = warp / 4 % 2, part = warp % 4, row = 32 * part + lane;
    const uint32_t lanes = static_cast<uint32_t>(32 * part) << 16;
    const uint32_t mine = tmem + 128 * t + 64 * half + lanes, result = tmem + o_column + 128 * t + half * (kDim / 2) + lanes;
    if (t < rows) {
      const float c = p.scale * kLog2e;
      float top = -INFINITY, total = 0;
#pragma unroll 1
      for (int j = 0; j < n; j++) {
        uint32_t s[64];
        warp_wait(s_full + 8 * t, j & 1, &failed);
        tmem_after_sync();
        load_scores(mine, s);
        if (partial(j)) {
          const int r = ring_of(j) % kMaskRing;
          warp_wait(masked + 8 * r, ring_of(j) / kMaskRing & 1, &failed);
          const uint32_t word0 = mask_words[r][2 * half], word1 = mask_words[r][2 * half + 1];
          if ((word0 & word1) != ~0u) mask_scores(word0, word1, s);
        }
        // what lay in `exchange` has been read: these scores were worked out after the other thread's weights of the tile before
        float now = most_of(s);
        exchange[t][half][row] = now;
        asm volatile("bar.sync %0, 64;" : : "r"(1 + 4 * t + part) : "memory");
        now = fmaxf(now, exchange[t][half ^ 1][row]);
        if (j == 0) {
          top = now;
        } else {
          const bool grows = (now - top) * c > kSlack;   // also from -infinity; not where both are
          if (__any_sync(~0u, grows)) {
            const float keep = grows ? exp2_of((top - now) * c) : 1.0f;
            if (grows) top = now;
            total *= keep;
            // this thread's half of the results; the products of tile j - 1 were done before the scores of tile j
#pragma unroll 1
            for (int x = 0; x < kDim / 2; x += 16) {
              uint32_t o[16];
              tmem_load<16>(result + x, o);
              tmem_loaded(o);
#pragma unroll
              for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
              tmem_store<16>(result + x, o);
            }
          }
        }
        const float base = top == -INFINITY ? 0.0f : -top * c;
        float2 sum[2] = {};
        weigh<T>(s, c, base, sum, mine);
        sum[0] = add2(sum[0], sum[1]);
        total += sum[0].x + sum[0].y;
        tmem_stored();
        tmem_before_sync();
        warp_arrive(p_full + 8 * t, lane);
      }
      const bool done = !n || warp_wait(o_full + 8 * t, 0, &failed);
      exchange[t][half][row] = total;
      asm volatile("bar.sync %0, 64;" : : "r"(1 + 4 * t + part) : "memory");
      total += exchange[t][half ^ 1][row];
      if (done) {
        tmem_after_sync();
        // only a sum of 0 is a row without keys; one that is not a number stays so, in lse too
        const float by = total == 0 ? 0.0f : 1.0f / total;
        const uint32_t staged = tiles_at + t * S::kTile;   // the queries are no longer needed
#pragma unroll
        for (int x = 0; x < kDim / 2; x += 32) {
          uint32_t o[32] = {};
          if (n) {
            tmem_load<32>(result + x, o);
            tmem_loaded(o);
          }
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = pack2<T>(__uint_as_float(o[k + 2 * i]) * by, __uint_as_float(o[k + 2 * i + 1]) * by);
            const int column = half * (kDim / 2) + x + k;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         : : "r"(staged + column / 64 * kBoxBytes + row * 128 + ((column % 64 / 8 ^ (row & 7)) * 16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          }
        }
        if (p.lse && half == 0 && q0 + 128 * t + row < p.q_tokens) {
          p.lse[(static_cast<int64_t>(batch) * p.q_heads + head) * p.q_tokens + q0 + 128 * t + row] =
              total == 0 ? -INFINITY : top * p.scale + logf(total);
        }
        fence_async_proxy();
        warp_arrive(staged_full + 8 * t, lane);
        if (row == 0 && half == 0 && barrier_wait(staged_full + 8 * t, 0, &failed)) {
          for (int x = 0; x < S::kBoxes && 64 * x < p.head_dim; x++) tile_store(&maps.out, 64 * x, q0 + 128 * t, head, batch, staged + x * kBoxBytes);
          tile_stores_read();
        }
      }
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 17) tmem_free<512>(tmem);
  if (failed) {
    const int3 at = rows_of(block_again());
    const int end = min(at.x + 256, p.q_tokens);
    spoil_rows(p.out, at.z, at.y, at.x, end, p.head_dim);
    for (int i = at.x + static_cast<int>(threadIdx.x); p.lse && i < end; i += kThreads) {
      p.lse[(static_cast<int64_t>(at.z) * p.q_heads + at.y) * p.q_tokens + i] = NAN;
    }
    if (threadIdx.x == 0) *p.status = 1;
  }
}

template <class T, int kDim>
cudaError_t launch(const CrossParams& p, const CrossMaps& maps, cudaStream_t stream) {
  constexpr int bytes = Sizes<kDim>::kShared;
  const cudaError_t e = allow_shared<cross_forward_kernel<T, kDim>>(bytes, p.device);
  if (e != cudaSuccess) return e;
  const unsigned blocks = static_cast<unsigned>((p.q_tokens + 255) / 256) * p.q_heads * p.batch;
  cross_forward_kernel<T, kDim><<<blocks, kThreads, bytes, stream>>>(p, maps);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cross_forward(const CrossParams& p, const CrossMaps& maps, int dtype, cudaStream_t stream) {
  if (dtype == MLXD_F16) return p.head_dim > 64 ? launch<__half, 128>(p, maps, stream) : launch<__half, 64>(p, maps, stream);
  return p.head_dim > 64 ? launch<__nv_bfloat16, 128>(p, maps, stream) : launch<__nv_bfloat16, 64>(p, maps, stream);
}

}  // namespace mlxd
