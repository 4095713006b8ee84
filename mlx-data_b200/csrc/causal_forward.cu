// Cached and window attention, forward: tiles of 128 rows against tiles of 128 keys on the tensor cores.
//
// One pass over the keys with a running maximum m and sum l of each row: S = Q K^T, P = 2^(c S - c m) with c = scale log2(e), O = O + P V,
// O and l scaled where m moves; at last O / l.  A tile's rows are tokens and the query heads that share a key head, head by head within a
// token, so that single tokens and short trees fill a tile as far as their heads go and keys are read once for all of them.  A CTA
// goes through the tiles of keys that its rows read: those of the first tokens that stay visible, then those of the window.  Keys of a
// cache come page by page.  Where rows are few, keys are split among CTAs, and within a CTA between its two halves; a second kernel
// joins the parts.
#include <algorithm>

#include "causal.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kThreads = 640;          // four warpgroups of softmax, then warps for copies, products, masks
constexpr int kMaskRing = 4;           // tiles of values in the ring are no more
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;         // as in cross attention: a row's reference maximum moves where its weight has grown by more than 2^8
constexpr int kByFma = 1;              // of eight pairs of exponentials, as there

template <int kDim>
struct Sizes {
  static constexpr int kTile = 128 * kDim * 2;             // bytes of 128 tokens
  static constexpr int kBoxes = kDim / 64;
  static constexpr int kSlots = kDim == 128 ? 5 : 8;       // of the ring of keys and values
  static constexpr int kShared = (2 + kSlots) * kTile;
};

__device__ __forceinline__ void load_scores(uint32_t at, uint32_t (&s)[64]) {
  tmem_load<32>(at, s);
  tmem_load<32>(at + 32, s + 32);
  tmem_loaded(s);
}

// -infinity where a key is not read.
__device__ __forceinline__ void mask_scores(uint64_t read, uint32_t (&s)[64]) {
  const uint32_t word0 = static_cast<uint32_t>(read), word1 = static_cast<uint32_t>(read >> 32);
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

// All of up to three barriers, 0 for none; one look at them where they are ready.
__device__ __forceinline__ bool warp_wait_all(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, uint32_t bar2, uint32_t parity2, volatile int* failed) {
  const bool a = !bar0 || barrier_try(bar0, parity0), b = !bar1 || barrier_try(bar1, parity1), c = !bar2 || barrier_try(bar2, parity2);
  if (__all_sync(~0u, a && b && c)) return true;
  return (!bar0 || warp_wait(bar0, parity0, failed)) && (!bar1 || warp_wait(bar1, parity1, failed)) && (!bar2 || warp_wait(bar2, parity2, failed));
}

// What a CTA does: up to two tiles of rows from token q0 on, or one in halves, of a key head's query heads, and which part of the keys.
struct Job {
  int q0, chunk, kv_head, batch, split;
};

// The last tiles of rows first: without a window they have the most keys.
template <class F>
__device__ __forceinline__ Job job_of(const F& f, int id) {
  const CausalParams& p = f.p;
  const int step = f.halves ? 1 : 2, tiles = (f.rows.tiles + step - 1) / step;
  Job j;
  j.kv_head = id % p.kv_heads;
  id /= p.kv_heads;
  j.split = id % f.splits;
  id /= f.splits;
  j.batch = id % p.batch;
  id /= p.batch;
  j.chunk = id % f.rows.chunks;
  j.q0 = (tiles - 1 - id / f.rows.chunks) * step * f.rows.tokens;
  return j;
}

template <class T, int kDim, bool kPaged>
__global__ void __launch_bounds__(kThreads, 1) causal_forward_kernel(const __grid_constant__ ForwardParams f, const __grid_constant__ CausalMaps maps) {
  using S = Sizes<kDim>;
  const CausalParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[2 + 2 * S::kSlots + 6 + 2 * kMaskRing + 2 + 1];
  __shared__ uint32_t mask_words[kMaskRing][4];
  __shared__ float exchange[2][2][128];   // of a row's two threads: maxima, sums at last
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, holes, first_place[2];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t tiles_at = smem_address(shared), ring_at = tiles_at + 2 * S::kTile;
  const uint32_t q_full = smem_address(bars), full = q_full + 16, empty = full + 8 * S::kSlots, s_full = empty + 8 * S::kSlots,
                 p_full = s_full + 16, o_full = p_full + 16, masked = o_full + 16, landed = masked + 8 * kMaskRing, staged_full = landed + 8 * kMaskRing, ended = staged_full + 16;
  const Job job = job_of(f, blockIdx.x);
  const int batch = job.batch, kv_head = job.kv_head, tile_tokens = f.rows.tokens, tile_heads = f.rows.heads;
  const Sequence seq = sequence_of<kPaged>(p, batch);
  if (threadIdx.x == 0) {
    failed = holes = 0;
    first_place[0] = first_place[1] = INT32_MAX;
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
  const uint32_t tmem = tmem_slot, o_column = 256;   // scores of tile t in columns 128 t, results in 256 + 128 t

  // ---------------------------------------------------- rows: this thread's, where it is one of the softmax
  const int t = warp / 8, half = warp / 4 % 2, part = warp % 4, row = 32 * part + lane;
  const int row_token = job.q0 + (f.halves ? 0 : t * tile_tokens) + row / tile_heads, in_group = job.chunk * tile_heads + row % tile_heads;
  const bool there = warp < 16 && row < tile_heads * tile_tokens && row_token < p.tokens && in_group < p.group;   // the row is in the result
  const bool reads = there && row_token < seq.fresh;
  Reach mine = {0, 0, 0};
  const uint8_t* tree = nullptr;
  if (reads) {
    int place = seq.held + row_token, to = min(place + 1, seq.end);
    if (p.tree) {
      tree = p.tree + batch * p.tree_batch + row_token * p.tree_token;
      place = seq.held;
      to = min(seq.held, seq.end);
      for (int j = 0; j < seq.fresh; j++) place += j != row_token && tree[j];
    }
    mine = reach_of(p, seq, place, to);
    if (p.tree) atomicMin(&first_place[t], place);
  }
  if (p.tree) __syncthreads();
  // what the rows of tile u read, in tiles of keys: those below `sinks`, and `from` to `to` - 1
  const auto reach_of_tile = [&](int u) {
    const int first = job.q0 + (f.halves ? 0 : u * tile_tokens), end = min(min(first + tile_tokens, p.tokens), seq.fresh);
    if (first >= end) return Reach{0, 0, 0};
    if (!p.tree) return reach_of(p, seq, seq.held + first, min(seq.held + end, seq.end));
    Reach a = reach_of(p, seq, first_place[f.halves ? 0 : u], seq.end);
    a.from = min(a.from, min(seq.held, seq.end));   // the new tokens are read by the tree alone
    a.sinks = min(a.sinks, a.from);
    return a;
  };
  const int row_tiles = f.halves || p.tokens - job.q0 <= tile_tokens ? 1 : 2;
  const Reach of_tile[2] = {reach_of_tile(0), f.halves ? reach_of_tile(0) : row_tiles == 2 ? reach_of_tile(1) : Reach{0, 0, 0}};
  // of the CTA: tile 0 begins first, tile 1 ends last, where it reads at all
  Reach all = of_tile[0];
  if (of_tile[1].to > of_tile[1].from || of_tile[1].sinks) {
    if (all.to > all.from || all.sinks) {
      all.from = min(all.from, of_tile[1].from);
      all.to = max(all.to, of_tile[1].to);
      all.sinks = min(max(all.sinks, of_tile[1].sinks), all.from);
    } else {
      all = of_tile[1];
    }
  }
  // the list of tiles of keys: first ones, then the window's; this CTA has `first` to `first` + n - 1 of it
  const int sink_tiles = (all.sinks + 127) / 128, main_first = max(all.from / 128, sink_tiles), main_end = all.to > all.from ? (all.to + 127) / 128 : 0;
  const int whole = sink_tiles + max(main_end - main_first, 0), share = (whole + f.splits - 1) / f.splits;
  const int first = min(job.split * share, whole), n = min(share, whole - first);
  const auto tile_of = [&](int j) { return j + first < sink_tiles ? j + first : j + first - sink_tiles + main_first; };
  const auto active = [&](int u, int j) {
    if (f.halves) return (j & 1) == u;
    const int tile = tile_of(j);
    const Reach& r = of_tile[u];
    return tile * 128 < r.sinks || (tile * 128 < r.to && tile * 128 + 128 > r.from && r.to > r.from);
  };
  // a tile whose keys are not all read by some row
  const auto partial = [&](int j) {
    const int lo = tile_of(j) * 128, hi = lo + 128;
    return holes || !(hi <= all.sinks || (lo >= all.from && hi <= all.to));
  };
  if (kPaged) {   // pages that are none, among those that are read
    const int entries = max(128 >> p.cache.page_shift, 1), wide = max(p.cache.page_shift - 7, 0);
    for (int e = threadIdx.x; e < n * entries; e += kThreads) {
      const int tile = tile_of(e / entries), entry = entries > 1 ? tile * entries + e % entries : tile >> wide;
      const int place = max(entry << p.cache.page_shift, tile * 128), end = min((entry + 1) << p.cache.page_shift, tile * 128 + 128);
      const bool needed = place < all.sinks || (place < all.to && end > all.from);
      if (needed && (entry >= p.cache.table_width || page_at(p.cache, batch, entry) < 0)) holes = 1;
    }
    __syncthreads();
  }

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 16 && n) {
      // -------------------------------------------------- copies: a lane has a page's box, or all of a tile's; lane 0 waits
      const int q_tiles = f.halves ? 1 : row_tiles;
      if (lane == 0) {
        for (int u = 0; u < q_tiles; u++) {
          barrier_expect(q_full + 8 * u, S::kBoxes * tile_heads * tile_tokens * 128);
          for (int x = 0; x < S::kBoxes; x++) {
            tile_load(tiles_at + u * S::kTile + x * kBoxBytes, &maps.q, 64 * x, job.chunk * tile_heads, job.q0 + u * tile_tokens, kv_head, batch, q_full + 8 * u);
          }
        }
      }
      const int pages = kPaged ? max(128 >> p.cache.page_shift, 1) : 1, x = lane / pages, page = lane % pages;   // of a tile; this lane's
      const bool copies = x < S::kBoxes;
      const auto major_of = [&](int j) {
        if (!kPaged) return batch;
        const int place = tile_of(j) * 128 + (page << (pages > 1 ? p.cache.page_shift : 0));
        return j < n && copies && place < p.cache.capacity ? page_of(p.cache, batch, place) : -1;
      };
      int issued = 0, partials = 0, major = major_of(0);
      bool going = true;
      for (; issued < 2 * n; issued++) {   // keys of tile 0, values of tile 0, keys of tile 1, ...
        const int slot = issued % S::kSlots, use = issued / S::kSlots, j = issued / 2;
        if (use) going = warp_wait(empty + 8 * slot, (use - 1) & 1, &failed);
        if (!going) break;
        // values of a tile that is not read as a whole go by way of the mask warp
        const bool by_masks = issued & 1 && partial(j);
        const uint32_t bar = by_masks ? landed + 8 * (partials % kMaskRing) : full + 8 * slot;
        if (lane == 0) barrier_expect(bar, S::kTile);
        __syncwarp();
        if (copies) {
          const int minor = kPaged ? (pages > 1 ? 0 : (tile_of(j) * 128) & (p.cache.page_size - 1)) : tile_of(j) * 128;
          tile_load(ring_at + slot * S::kTile + x * kBoxBytes + page * (kBoxBytes / pages), issued & 1 ? &maps.v : &maps.k, 64 * x, minor, kv_head, major, bar);
        }
        if (issued & 1) {
          partials += by_masks;
          major = major_of(j + 1);
        }
      }
      if (!going && lane == 0) {   // what is under way still lands before the CTA ends
        for (int u = 0; u < q_tiles; u++) {
          for (int i = 0; i < kWaitTries && !barrier_try(q_full + 8 * u, 0); i++) {}
        }
        int r = 0;
        for (int k = 0; k < issued; k++) {
          const bool by_masks = k & 1 && partial(k / 2);
          const uint32_t bar = by_masks ? landed + 8 * (r % kMaskRing) : full + 8 * (k % S::kSlots);
          const uint32_t parity = (by_masks ? r / kMaskRing : k / S::kSlots) & 1;
          r += by_masks;
          if (k < issued - S::kSlots) continue;
          for (int i = 0; i < kWaitTries && !barrier_try(bar, parity); i++) {}
        }
      }
    } else if (warp == 17 && n) {
      // -------------------------------------------------- products
      constexpr uint32_t kScores = product_descriptor<T>(128, 128, false), kResults = product_descriptor<T>(128, kDim, true);
      const int steps = (p.head_dim + 15) / 16, users = f.halves ? 2 : row_tiles;
      const uint32_t queries = low_half(at_address(tile_descriptor(16), tiles_at)), keys = low_half(at_address(tile_descriptor(16), ring_at)),
                     values = low_half(at_address(tile_descriptor(kBoxBytes), ring_at));
      const auto scores = [&](int u, uint32_t slot) {   // S = Q K^T
        product_of_tiles<kDim>(tmem + 128 * u, queries + (f.halves ? 0 : u * (S::kTile >> 4)), keys + slot * (S::kTile >> 4), kScores, steps);
        products_done(s_full + 8 * u);
      };
      Ring<S::kSlots> at;                               // the item that is needed next
      bool going = warp_wait(full, 0, &failed);
      for (int u = 0; u < users && going; u++) {
        if (!f.halves || u == 0) going = warp_wait(q_full + 8 * u, 0, &failed);
        if (going && elected()) {
          if (active(u, 0)) scores(u, 0);
          if (u + 1 == users) products_done(empty + 0);
        }
        __syncwarp();
      }
      at.next();
      // The tensor cores run a product or two behind the thread that issues them, so between two groups of products there is one
      // look at barriers and no more: with the last group of a tile of keys, at those of the next one's tiles too.
      Ring<S::kSlots> v = at, k = at;
      k.next();
      going = going && warp_wait_all(full + 8 * v.slot, v.phase, n > 1 ? full + 8 * k.slot : 0, k.phase, 0, 0, &failed);
      uint32_t done[2] = {0, 0};                        // tiles of keys that each tile of rows has taken
      int last_of[2] = {n - 1, n - 1};                  // the last one
      for (int u = 0; u < users; u++) {
        while (last_of[u] >= 0 && !active(u, last_of[u])) last_of[u]--;
      }
#pragma unroll 1
      for (int j = 0; j < n && going; j++) {
        Ring<S::kSlots> next_v = k, next_k;
        next_v.next();
        next_k = next_v;
        next_k.next();
#pragma unroll
        for (int u = 0; u < 2; u++) {
          if (u >= users || !going) break;
          // O += P V, P where the scores were, when both halves of the keys have been weighed
          const uint32_t o = tmem + o_column + 128 * u, values_at = values + v.slot * (S::kTile >> 4);
          const bool last = u + 1 == users, weighs = active(u, j), more = j + 1 < n && active(u, j + 1);
          going = warp_wait_all(weighs ? p_full + 8 * u : 0, done[u] & 1, last && j + 1 < n ? full + 8 * next_v.slot : 0, next_v.phase,
                                last && j + 2 < n ? full + 8 * next_k.slot : 0, next_k.phase, &failed);
          if (!going) break;
          tmem_after_sync();
          if (elected()) {
            if (weighs) {
              product_over_tokens(o, tmem + 128 * u, values_at, kResults, done[u] > 0);
              product_over_tokens(o, tmem + 128 * u + 64, values_at + kHalfTokens, kResults, true);
              if (j == last_of[u]) products_done(o_full + 8 * u);
            }
            if (last) products_done(empty + 8 * v.slot);
            // products run in the order in which they are issued: these scores overwrite P after it has been read
            if (more) scores(u, k.slot);
            if (last && j + 1 < n) products_done(empty + 8 * k.slot);
          }
          __syncwarp();
          done[u] += weighs;
        }
        v = next_v;
        k = next_k;
      }
      if (!going) products_end(ended);
    } else if (warp == 19) {
      // -------------------------------------------------- masks: which keys are read, and zeros where values are not
      int r = 0;
      for (int j = 0; j < n; j++) {
        if (!partial(j)) continue;
        uint32_t words[4];
        for (int i = 0; i < 4; i++) {
          const int key = tile_of(j) * 128 + i * 32 + lane;
          bool read = key < all.sinks || (key >= all.from && key < all.to);
          if (kPaged && read && holes) read = page_of(p.cache, batch, key) >= 0;
          words[i] = __ballot_sync(~0u, read);
        }
        const int item = 2 * j + 1;
        if (!warp_wait(landed + 8 * (r % kMaskRing), r / kMaskRing & 1, &failed)) break;
        const uint32_t values = ring_at + item % S::kSlots * S::kTile;
        for (int i = 0; i < 4; i++) {
          if (lane == 0) mask_words[r % kMaskRing][i] = words[i];
          // 8 lanes a row of 128 bytes
          for (int v = lane / 8; v < 32; v += 4) {
            if (words[i] >> v & 1) continue;
            for (int x = 0; x < S::kBoxes; x++) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                           : : "r"(values + x * kBoxBytes + (32 * i + v) * 128 + (lane & 7) * 16), "r"(0) : "memory");
            }
          }
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) {
          barrier_arrive(full + 8 * (item % S::kSlots));
          barrier_arrive(masked + 8 * (r % kMaskRing));
        }
        r++;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------------------------------------------- softmax: a row belongs to two threads, one for each half of the keys of a tile
    // A wait that ran out does not end the loop: the two warps of a row's threads meet at a barrier for every tile.
    const uint32_t lanes = static_cast<uint32_t>(32 * part) << 16;
    const uint32_t scores_at = tmem + 128 * t + 64 * half + lanes, result = tmem + o_column + 128 * t + half * (kDim / 2) + lanes;
    if (f.halves || t < row_tiles) {
      const float c = p.scale * kLog2e;
      float top = -INFINITY, total = 0;
      int done = 0;
#pragma unroll 1
      for (int j = 0; j < n; j++) {
        if (!active(t, j)) continue;
        uint32_t s[64];
        warp_wait(s_full + 8 * t, done & 1, &failed);
        tmem_after_sync();
        load_scores(scores_at, s);
        const int first_key = tile_of(j) * 128 + 64 * half;
        const bool whole_tile = (first_key >= mine.from && first_key + 64 <= mine.to) || first_key + 64 <= mine.sinks;
        if (!__all_sync(~0u, whole_tile) || holes) {
          uint64_t read = bits_of(first_key, mine.from, mine.to) | bits_of(first_key, 0, mine.sinks);
          if (tree) {
            for (int k = max(first_key, seq.held); k < min(first_key + 64, seq.end); k++) {
              if (tree[k - seq.held]) read |= uint64_t{1} << (k - first_key);
            }
          }
          if (holes) {
            warp_wait(masked + 8 * (j % kMaskRing), j / kMaskRing & 1, &failed);
            const uint32_t* words = mask_words[j % kMaskRing] + 2 * half;
            read &= words[0] | static_cast<uint64_t>(words[1]) << 32;
          }
          mask_scores(read, s);
        }
        // what lay in `exchange` has been read: these scores were worked out after the other thread's weights of the tile before
        float now = most_of(s);
        exchange[t][half][row] = now;
        asm volatile("bar.sync %0, 64;" : : "r"(1 + 4 * t + part) : "memory");
        now = fmaxf(now, exchange[t][half ^ 1][row]);
        if (done == 0) {
          top = now;
        } else {
          const bool grows = (now - top) * c > kSlack;   // also from -infinity; not where both are
          if (__any_sync(~0u, grows)) {
            const float keep = grows ? exp2_of((top - now) * c) : 1.0f;
            if (grows) top = now;
            total *= keep;
            // this thread's half of the results; the products of the tile before were done before these scores
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
        weigh<T>(s, c, base, sum, scores_at);
        sum[0] = add2(sum[0], sum[1]);
        total += sum[0].x + sum[0].y;
        tmem_stored();
        tmem_before_sync();
        warp_arrive(p_full + 8 * t, lane);
        done++;
      }
      const bool valid = !done || warp_wait(o_full + 8 * t, 0, &failed);
      exchange[t][half][row] = total;
      asm volatile("bar.sync %0, 64;" : : "r"(1 + 4 * t + part) : "memory");
      total += exchange[t][half ^ 1][row];
      if (valid) {
        tmem_after_sync();
        // only a sum of 0 is a row without keys; one that is not a number stays so, in lse too
        const float by = total == 0 ? 0.0f : 1.0f / total;
        const float lse = total == 0 ? -INFINITY : top * p.scale + logf(total);
        const int64_t stat = (static_cast<int64_t>(batch) * p.q_heads + kv_head * p.group + in_group) * p.tokens + row_token;
        const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.tokens, slot = f.halves ? 2 * job.split + t : job.split;
        const uint32_t staged = tiles_at + t * S::kTile;   // the queries are no longer needed
        const bool any = __any_sync(~0u, total != 0);
#pragma unroll
        for (int x = 0; x < kDim / 2; x += 32) {
          uint32_t o[32] = {};
          if (done) {
            tmem_load<32>(result + x, o);
            tmem_loaded(o);
          }
          if (f.parts > 1) {
            if (there && total != 0) {   // a part without keys is not read when they are joined
              float* to = f.part_out + (slot * rows + stat) * p.head_dim + half * (kDim / 2) + x;
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                if (half * (kDim / 2) + x + k < p.head_dim) {
                  *reinterpret_cast<float4*>(to + k) = make_float4(__uint_as_float(o[k]) * by, __uint_as_float(o[k + 1]) * by, __uint_as_float(o[k + 2]) * by, __uint_as_float(o[k + 3]) * by);
                }
              }
            }
            continue;
          }
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              // what a row without keys has summed is nothing, whatever stands there
              w[i] = any && total != 0 ? pack2<T>(__uint_as_float(o[k + 2 * i]) * by, __uint_as_float(o[k + 2 * i + 1]) * by) : 0u;
            }
            const int column = half * (kDim / 2) + x + k;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         : : "r"(staged + column / 64 * kBoxBytes + row * 128 + ((column % 64 / 8 ^ (row & 7)) * 16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          }
        }
        if (half == 0 && there) {
          if (f.parts > 1) f.part_lse[slot * rows + stat] = lse;
          else if (p.lse) p.lse[stat] = lse;
        }
        if (f.parts == 1) {
          fence_async_proxy();
          warp_arrive(staged_full + 8 * t, lane);
          if (row == 0 && half == 0 && barrier_wait(staged_full + 8 * t, 0, &failed)) {
            for (int x = 0; x < S::kBoxes && 64 * x < p.head_dim; x++) {
              tile_store(&maps.out, 64 * x, job.chunk * tile_heads, job.q0 + t * tile_tokens, kv_head, batch, staged + x * kBoxBytes);
            }
            tile_stores_read();
          }
        }
      }
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 17) tmem_free<512>(tmem);
  if (failed) {   // not a number, instead of whatever the memory held
    const Job at = job_of(f, block_again());
    const int step = f.halves ? 1 : 2, rows = step * f.rows.tokens * f.rows.heads;
    for (int i = threadIdx.x / 32; i < rows; i += kThreads / 32) {
      const int token = at.q0 + i / f.rows.heads, head = at.chunk * f.rows.heads + i % f.rows.heads;
      if (token >= p.tokens || head >= p.group) continue;
      const int64_t stat = (static_cast<int64_t>(at.batch) * p.q_heads + at.kv_head * p.group + head) * p.tokens + token;
      if (f.parts > 1) {
        for (int u = 0; u < (f.halves ? 2 : 1); u++) {
          const int64_t part_row = (f.halves ? 2 * at.split + u : at.split) * static_cast<int64_t>(p.batch) * p.q_heads * p.tokens + stat;
          for (int e = lane; e < p.head_dim; e += 32) f.part_out[part_row * p.head_dim + e] = NAN;
          if (lane == 0) f.part_lse[part_row] = NAN;
        }
      } else {
        uint16_t* to = reinterpret_cast<uint16_t*>(p.out.data) + at.batch * p.out.batch + token * p.out.token + (at.kv_head * p.group + head) * p.out.head;
        for (int e = lane; e < p.head_dim; e += 32) to[e] = 0x7fff;
        if (p.lse && lane == 0) p.lse[stat] = NAN;
      }
    }
    if (threadIdx.x == 0) *p.status = 1;
  }
}

// The parts of a row, weighted by exp(lse): a warp a row, four elements a lane.
constexpr int kJoinWarps = 4;

template <class T>
__global__ void __launch_bounds__(32 * kJoinWarps) causal_join_kernel(const __grid_constant__ ForwardParams f) {
  const CausalParams& p = f.p;
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.tokens, stat = static_cast<int64_t>(blockIdx.x) * kJoinWarps + threadIdx.x / 32;
  if (stat >= rows) return;
  const int token = stat % p.tokens, head = stat / p.tokens % p.q_heads, batch = stat / p.tokens / p.q_heads;
  wait_for_kernels_before();
  float top = -INFINITY;
  for (int i = lane; i < f.parts; i += 32) top = max_or_nan(top, f.part_lse[i * rows + stat]);
  for (int d = 16; d; d >>= 1) top = max_or_nan(top, __shfl_xor_sync(~0u, top, d));
  float4 o = {};
  float total = 0;
  const bool there = 4 * lane < p.head_dim;
  if (top != -INFINITY) {
    for (int i0 = 0; i0 < f.parts; i0 += 32) {
      const float w = i0 + lane < f.parts ? exp2_of((f.part_lse[(i0 + lane) * rows + stat] - top) * kLog2e) : 0.0f;
      const int end = min(32, f.parts - i0);
#pragma unroll 4
      for (int i = 0; i < end; i++) {
        const float wi = __shfl_sync(~0u, w, i);
        if (wi == 0.0f) continue;    // also a part without keys, where nothing was written
        const float4 x = there ? *reinterpret_cast<const float4*>(f.part_out + ((i0 + i) * rows + stat) * p.head_dim + 4 * lane) : make_float4(0, 0, 0, 0);
        total += wi;
        o.x += wi * x.x;
        o.y += wi * x.y;
        o.z += wi * x.z;
        o.w += wi * x.w;
      }
    }
  }
  const float by = total == 0 ? 0.0f : 1.0f / total;
  if (there) {
    T* to = reinterpret_cast<T*>(p.out.data) + batch * p.out.batch + token * p.out.token + head * p.out.head + 4 * lane;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(o.x * by, o.y * by), pack2<T>(o.z * by, o.w * by));
  }
  if (lane == 0 && p.lse) p.lse[stat] = total == 0 ? -INFINITY : top + logf(total);
}

template <class T, int kDim, bool kPaged>
cudaError_t launch(const ForwardParams& f, const CausalMaps& maps, cudaStream_t stream) {
  constexpr int bytes = Sizes<kDim>::kShared;
  const CausalParams& p = f.p;
  const cudaError_t e = allow_shared<causal_forward_kernel<T, kDim, kPaged>>(bytes, p.device);
  if (e != cudaSuccess) return e;
  const int step = f.halves ? 1 : 2;
  const unsigned blocks = static_cast<unsigned>((f.rows.tiles + step - 1) / step) * f.rows.chunks * f.splits * p.kv_heads * p.batch;
  causal_forward_kernel<T, kDim, kPaged><<<blocks, kThreads, bytes, stream>>>(f, maps);
  return cudaGetLastError();
}

template <class T>
cudaError_t launch_join(const ForwardParams& f, cudaStream_t stream) {
  const CausalParams& p = f.p;
  // begins while the parts are being worked out and waits for them on the device
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.batch) * p.q_heads * p.tokens + kJoinWarps - 1) / kJoinWarps));
  config.blockDim = dim3(32 * kJoinWarps);
  config.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, causal_join_kernel<T>, f);
}

template <class T, int kDim>
cudaError_t launch(const ForwardParams& f, const CausalMaps& maps, bool paged, cudaStream_t stream) {
  return paged ? launch<T, kDim, true>(f, maps, stream) : launch<T, kDim, false>(f, maps, stream);
}

}  // namespace

ForwardParams forward_plan(const CausalParams& p, bool paged, int sms) {
  ForwardParams f = {};
  f.p = p;
  f.rows = row_tiles(p);
  f.splits = f.cluster = 1;
  const int64_t sixteens = (static_cast<int64_t>(p.tokens) * p.group + 15) / 16, heads = static_cast<int64_t>(p.batch) * p.kv_heads;
  f.steps = paged && sixteens <= 1 && p.kv_heads <= 65535 && p.batch * int64_t{64} <= 65535;
  f.halves = paged && !f.steps && f.rows.tiles == 1;
  if (f.steps) {
    int64_t reach = p.cache.capacity;
    if (p.window != INT32_MAX) reach = std::min(reach, static_cast<int64_t>(p.window) + p.tokens + std::min(p.sinks, p.cache.capacity) + 32);
    const int64_t rounds = std::max<int64_t>(1, reach / 64);    // of a CTA's four warps
    const int64_t slots = static_cast<int64_t>(step_ctas(p.head_dim, p.tokens * p.group <= 8 ? 1 : 2)) * sms;
    while (f.cluster < 8 && 2 * heads * f.cluster <= slots && f.cluster * 2 <= rounds) f.cluster *= 2;
    f.splits = static_cast<int>(std::max<int64_t>(1, std::min({reach / (f.cluster * 1500), 8 * slots / (heads * f.cluster), int64_t{64}})));
    f.parts = f.splits;
    return f;
  }
  const int64_t ctas = static_cast<int64_t>((f.rows.tiles + (f.halves ? 0 : 1)) / (f.halves ? 1 : 2)) * f.rows.chunks * p.batch * p.kv_heads;
  if (paged) {
    // tiles of keys that a CTA may have
    int64_t most = (p.cache.capacity + 127) / 128;
    if (p.window != INT32_MAX) most = std::min(most, (static_cast<int64_t>(p.window) + 2 * f.rows.tokens + 127) / 128 + 1 + (std::min(p.sinks, p.cache.capacity) + 127) / 128);
    const int64_t want = f.halves ? 4 * sms : sms;
    f.splits = static_cast<int>(std::max<int64_t>(1, std::min(most, std::min<int64_t>(want / ctas, 64))));
  }
  f.parts = f.splits * (f.halves ? 2 : 1);
  return f;
}

size_t forward_workspace(const ForwardParams& f) {
  const CausalParams& p = f.p;
  return f.parts > 1 ? sizeof(float) * f.parts * p.batch * p.q_heads * p.tokens * (p.head_dim + 1) : 0;
}

cudaError_t launch_causal_join(const ForwardParams& f, int dtype, cudaStream_t stream) {
  return dtype == MLXD_F16 ? launch_join<__half>(f, stream) : launch_join<__nv_bfloat16>(f, stream);
}

cudaError_t launch_causal_forward(const ForwardParams& f, const CausalMaps& maps, bool paged, int dtype, cudaStream_t stream) {
  if (dtype == MLXD_F16) return f.p.head_dim > 64 ? launch<__half, 128>(f, maps, paged, stream) : launch<__half, 64>(f, maps, paged, stream);
  return f.p.head_dim > 64 ? launch<__nv_bfloat16, 128>(f, maps, paged, stream) : launch<__nv_bfloat16, 64>(f, maps, paged, stream);
}

}  // namespace mlxd
