// Cached and window attention, forward: tiles of 128 rows against tiles of 128 keys on the tensor cores.
//
// One pass over the keys with a running maximum m and sum l of each row: S = Q K^T, P = 2^(c S - c m) with c = scale log2(e), O = O + P V,
// O and l scaled where m moves; at last O / l.  A tile's rows are tokens and the query heads that share a key head, head by head within a
// token, so that single tokens and short trees fill a tile as far as their heads go and keys are read once for all of them.  A CTA
// goes through the tiles of keys that its rows read: those of the first tokens that stay visible, then those of the window.  Keys of a
// cache come page by page.  Where rows are few, keys are split among CTAs, and within a CTA between its two halves; a second kernel
// joins the parts.
//
// 4 D operations a pair of row and key, so the tensor cores are the floor of long calls; two tiles of rows take 2048 cycles of products for a
// tile of keys, and 3300 to 3600 as measured: products read both operands from shared memory, 128 bytes a cycle, which copies and
// exchanges share, and a tile's softmax (1600 to 1900 cycles) and products follow one another.  A job's first and last tiles, of which a
// part is masked, and its results cost about 4 us more.  Measured: 2 x 4099 tokens, 32 heads on 8 of 128, window 1024, 4 first tokens
// 173-178 us, 680 TFLOP/s (42 % of the measured rate); a chunk of 2048 tokens behind 6404 keys 268-277 us, 910; eight trees of 25 drafts
// over up to 8217 keys 68 us, 3.1 TB/s, of which CTAs stream for 36.  Stores of results by tile copies took 3000 to 6000 cycles a tile
// and held up the softmax, or, from a warp of their own, the next tile's: rows go from registers, 32 bytes a thread.
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
  // In halves there is one tile of queries, and a tile of heads of 128 more in the ring: keys two tiles ahead of the weights wait for no
  // values then (eight trees of 25 drafts, up to 8217 keys: 75.4 us with five places, 70.9 with six).
  static constexpr int kHalfSlots = kDim == 128 ? 6 : 8;
  static constexpr int kShared = (2 + kSlots) * kTile;     // and queries of two tiles
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

// A job: up to two tiles of rows from token q0 on, or one in halves, of a key head's query heads, and which part of the keys.
struct Job {
  int q0, chunk, kv_head, batch, split;
};

__host__ __device__ inline int64_t jobs_of(const ForwardParams& f) {
  const int step = f.halves ? 1 : 2;
  return static_cast<int64_t>((f.rows.tiles + step - 1) / step) * f.rows.chunks * f.splits * f.p.kv_heads * f.p.batch;
}

// The last tiles of rows first: without a window they have the most keys.
__device__ __forceinline__ Job job_of(const ForwardParams& f, int id) {
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

// What is to be done for a job, in tiles of 128 keys: those that its rows read are first ones and then the window's, and the job has n of
// this list from `first` on.
struct Work {
  Job job;
  Sequence seq;
  int row_tiles;
  Reach of[2], all;             // what the rows of each tile read, and of both
  int sink_tiles, main_first, first, n;

  __device__ __forceinline__ int tile(int j) const { return j + first < sink_tiles ? j + first : j + first - sink_tiles + main_first; }

  // Whether rows that read `r` read some key of tile j.
  __device__ __forceinline__ bool touches(const Reach& r, int j) const {
    const int lo = tile(j) * 128;
    return lo < r.sinks || (lo < r.to && lo + 128 > r.from && r.to > r.from);
  }

  // Whether values of tile j that no row reads need no clearing: there are none in a cache, or none behind the sequence, whose tensor's end
  // is zeros by itself.
  template <bool kPaged>
  __device__ __forceinline__ bool whole(int j, int tokens) const {
    const int lo = tile(j) * 128, hi = lo + 128;
    if (!kPaged) return hi <= seq.end || seq.end == tokens;
    return hi <= all.sinks || (lo >= all.from && hi <= all.to);
  }
};

// `first_place`: with a tree, the first place that the rows of each tile have.
template <bool kPaged>
__device__ __forceinline__ Work work_of(const ForwardParams& f, int id, const volatile int* first_place) {
  const CausalParams& p = f.p;
  Work w;
  w.job = job_of(f, id);
  w.seq = sequence_of<kPaged>(p, w.job.batch);
  w.row_tiles = f.halves || p.tokens - w.job.q0 <= f.rows.tokens ? 1 : 2;
  const auto reach_of_tile = [&](int u) {
    const int first = w.job.q0 + u * f.rows.tokens, end = min(min(first + f.rows.tokens, p.tokens), w.seq.fresh);
    if (first >= end) return Reach{0, 0, 0};
    if (!kPaged || !p.tree) return reach_of(p, w.seq, w.seq.held + first, min(w.seq.held + end, w.seq.end));
    Reach a = reach_of(p, w.seq, first_place[u], w.seq.end);
    a.from = min(a.from, min(w.seq.held, w.seq.end));   // the new tokens are read by the tree alone
    a.sinks = min(a.sinks, a.from);
    return a;
  };
  w.of[0] = reach_of_tile(0);
  w.of[1] = f.halves ? w.of[0] : reach_of_tile(1);
  // tile 0 begins first, tile 1 ends last, where it reads at all
  w.all = w.of[0];
  if (w.of[1].to > w.of[1].from || w.of[1].sinks) {
    w.all.from = min(w.all.from, w.of[1].from);
    w.all.to = max(w.all.to, w.of[1].to);
    w.all.sinks = min(max(w.all.sinks, w.of[1].sinks), w.all.from);
  }
  w.sink_tiles = (w.all.sinks + 127) / 128;
  w.main_first = max(w.all.from / 128, w.sink_tiles);
  const int whole = w.sink_tiles + (w.all.to > w.all.from ? max((w.all.to + 127) / 128 - w.main_first, 0) : 0);
  const int share = f.splits == 1 ? whole : (whole + f.splits - 1) / f.splits;
  w.first = min(w.job.split * share, whole);
  w.n = min(share, whole - w.first);
  return w;
}

// A CTA takes one job after another, every gridDim.x-th: copies and products of the next begin while the results of the one before are
// written (window attention; a cache has as many CTAs as jobs, since which of its pages are none is found by the whole CTA).
template <class T, int kDim, bool kPaged>
__global__ void __launch_bounds__(kThreads, 1) causal_forward_kernel(const __grid_constant__ ForwardParams f, const __grid_constant__ CausalMaps maps) {
  using S = Sizes<kDim>;
  const CausalParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ uint64_t bars[4 + 2 * S::kHalfSlots + 6 + 2 * kMaskRing + 1];
  __shared__ uint32_t mask_words[kMaskRing][4];
  __shared__ float exchange[2][2][128];   // of a row's two threads: maxima, sums at last
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, holes, first_place[2], gave_up[2][4];
  __shared__ uint32_t progress;           // copies begun
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const uint32_t tiles_at = smem_address(shared), ring_at = tiles_at + (f.halves && S::kHalfSlots > S::kSlots ? 1 : 2) * S::kTile;
  const uint32_t q_full = smem_address(bars), q_empty = q_full + 16, full = q_empty + 16, empty = full + 8 * S::kHalfSlots, s_full = empty + 8 * S::kHalfSlots,
                 p_full = s_full + 16, o_full = p_full + 16, masked = o_full + 16, landed = masked + 8 * kMaskRing, ended = landed + 8 * kMaskRing;
  const int tile_tokens = f.rows.tokens, tile_heads = f.rows.heads, jobs = static_cast<int>(jobs_of(f));
  const uint32_t slots = f.halves ? S::kHalfSlots : S::kSlots;
  if (threadIdx.x == 0) {
    failed = holes = 0;
    progress = 0;
    for (int i = 0; i < 8; i++) gave_up[i / 4][i % 4] = 0;
    first_place[0] = first_place[1] = INT32_MAX;
    barrier_init(ended, 1);
    for (int t = 0; t < 2; t++) {
      barrier_init(q_full + 8 * t, 1);
      barrier_init(q_empty + 8 * t, 1);
      barrier_init(s_full + 8 * t, 1);
      barrier_init(p_full + 8 * t, 8);
      barrier_init(o_full + 8 * t, 1);
    }
    for (int i = 0; i < S::kHalfSlots; i++) {
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
  wait_for_kernels_before();
  const uint32_t tmem = tmem_slot, o_column = 256;   // scores of tile t in columns 128 t, results in 256 + 128 t
  // ---------------------------------------------------- this thread's row, where it is one of the softmax
  const int t = warp / 8, half = warp / 4 % 2, part = warp % 4, row = 32 * part + lane;
  const int row_token = (f.halves ? 0 : t * tile_tokens) + row / tile_heads, row_head = row % tile_heads;
  int tree_place = 0;
  if (kPaged && p.tree) {   // a warp counts what a token reads; `exchange` is not needed yet
    const Job job = job_of(f, blockIdx.x);
    const Sequence seq = sequence_of<kPaged>(p, job.batch);
    int* const places = reinterpret_cast<int*>(exchange);
    for (int i = warp; i < (f.halves ? 1 : 2) * tile_tokens; i += kThreads / 32) {
      const int token = job.q0 + i;
      if (token >= seq.fresh) break;
      const uint8_t* tree = p.tree + job.batch * p.tree_batch + token * p.tree_token;
      int others = 0;
      for (int j = lane; j < seq.fresh; j += 32) others += j != token && tree[j];
      others = __reduce_add_sync(~0u, others);
      if (lane == 0) {
        places[i] = seq.held + others;
        atomicMin(&first_place[i / tile_tokens], seq.held + others);
      }
    }
    __syncthreads();
    if (warp < 16 && row < tile_heads * tile_tokens && job.q0 + row_token < seq.fresh) tree_place = places[row_token];
  }
  if (kPaged) {   // pages that are none, among those that are read
    const Work w = work_of<kPaged>(f, blockIdx.x, first_place);
    const int entries = max(128 >> p.cache.page_shift, 1), wide = max(p.cache.page_shift - 7, 0);
    for (int e = threadIdx.x; e < w.n * entries; e += kThreads) {
      const int tile = w.tile(e / entries), entry = entries > 1 ? tile * entries + e % entries : tile >> wide;
      const int place = max(entry << p.cache.page_shift, tile * 128), end = min((entry + 1) << p.cache.page_shift, tile * 128 + 128);
      const bool needed = place < w.all.sinks || (place < w.all.to && end > w.all.from);
      if (needed && (entry >= p.cache.table_width || page_at(p.cache, w.job.batch, entry) < 0)) holes = 1;
    }
    __syncthreads();
  }
  const bool gaps = kPaged && holes;

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 16) {
      // -------------------------------------------------- copies: a lane has a page's box, or all of a tile's; lane 0 waits
      const int pages = kPaged ? max(128 >> p.cache.page_shift, 1) : 1, x = lane / pages, page = lane % pages;   // of a tile; this lane's
      const bool copies = x < S::kBoxes;
      uint32_t issued = 0, partials = 0, queries[2] = {0, 0}, how = 0;   // how: four bits a slot, which barrier its copy goes to
      bool going = true;
      for (int id = blockIdx.x; id < jobs && going; id += gridDim.x) {
        const Work w = work_of<kPaged>(f, id, first_place);
        if (!w.n) continue;
#pragma unroll
        for (int u = 0; u < 2; u++) {
          if (u >= w.row_tiles || !going) break;
          if (queries[u]) going = warp_wait(q_empty + 8 * u, (queries[u] - 1) & 1, &failed);
          if (!going) break;
          if (lane == 0) {
            barrier_expect(q_full + 8 * u, S::kBoxes * tile_heads * tile_tokens * 128);
            for (int y = 0; y < S::kBoxes; y++) {
              tile_load(tiles_at + u * S::kTile + y * kBoxBytes, &maps.q, 64 * y, w.job.chunk * tile_heads, w.job.q0 + u * tile_tokens, w.job.kv_head, w.job.batch, q_full + 8 * u);
            }
          }
          queries[u]++;
        }
        const auto major_of = [&](int j) {
          if (!kPaged) return w.job.batch;
          const int place = w.tile(j) * 128 + (page << (pages > 1 ? p.cache.page_shift : 0));
          return j < w.n && copies && place < p.cache.capacity ? page_of(p.cache, w.job.batch, place) : -1;
        };
        int major = major_of(0);
        for (int i = 0; i < 2 * w.n && going; i++) {   // keys of tile 0, values of tile 0, keys of tile 1, ...
          const int j = i / 2;
          const uint32_t slot = issued % slots, use = issued / slots;
          if (use) going = warp_wait(empty + 8 * slot, (use - 1) & 1, &failed);
          if (!going) break;
          // values of a tile that is not read as a whole go by way of the mask warp
          const bool by_masks = i & 1 && (gaps || !w.template whole<kPaged>(j, p.tokens));
          const uint32_t bar = by_masks ? landed + 8 * (partials % kMaskRing) : full + 8 * slot;
          if (lane == 0) barrier_expect(bar, S::kTile);
          __syncwarp();
          how = (how & ~(15u << (4 * slot))) | ((by_masks ? 8 | (partials % (2 * kMaskRing)) : use & 1) << (4 * slot));
          if (copies) {
            const int minor = kPaged ? (pages > 1 ? 0 : (w.tile(j) * 128) & (p.cache.page_size - 1)) : w.tile(j) * 128;
            tile_load(ring_at + slot * S::kTile + x * kBoxBytes + page * (kBoxBytes / pages), i & 1 ? &maps.v : &maps.k, 64 * x, minor, w.job.kv_head, major, bar);
          }
          issued++;
          if (lane == 0) *static_cast<volatile uint32_t*>(&progress) = issued;
          if (i & 1) {
            partials += by_masks;
            major = major_of(j + 1);
          }
        }
      }
      if (!going && lane == 0) {   // what is under way still lands before the CTA ends
        for (int u = 0; u < 2; u++) {
          for (int i = 0; queries[u] && i < kWaitTries && !barrier_try(q_full + 8 * u, (queries[u] - 1) & 1); i++) {}
        }
        for (uint32_t k = 0; k < min(issued, slots); k++) {
          const uint32_t of = how >> (4 * k) & 15;
          const uint32_t bar = of & 8 ? landed + 8 * (of % kMaskRing) : full + 8 * k, parity = of & 8 ? of / kMaskRing & 1 : of;
          for (int i = 0; i < kWaitTries && !barrier_try(bar, parity); i++) {}
        }
      }
    } else if (warp == 17) {
      // -------------------------------------------------- products
      constexpr uint32_t kScores = product_descriptor<T>(128, 128, false), kResults = product_descriptor<T>(128, kDim, true);
      const int steps = (p.head_dim + 15) / 16;
      const uint32_t queries = low_half(at_address(tile_descriptor(16), tiles_at)), keys = low_half(at_address(tile_descriptor(16), ring_at)),
                     values = low_half(at_address(tile_descriptor(kBoxBytes), ring_at));
      const auto scores = [&](int u, uint32_t slot) {   // S = Q K^T
        product_of_tiles<kDim>(tmem + 128 * u, queries + (f.halves ? 0 : u * (S::kTile >> 4)), keys + slot * (S::kTile >> 4), kScores, steps);
        products_done(s_full + 8 * u);
      };
      Ring<S::kSlots> k;                                // the item that is needed next
      uint32_t done[2] = {0, 0}, loaded[2] = {0, 0};    // tiles of keys that each tile of rows has taken; its loads of queries
      bool going = true;
      for (int id = blockIdx.x; id < jobs && going; id += gridDim.x) {
        const Work w = work_of<kPaged>(f, id, first_place);
        if (!w.n) continue;
        const int n = w.n, users = w.row_tiles;
        const auto active = [&](int u, int j) { return w.touches(w.of[u], j); };
        if (f.halves) {
          // Tile j is the half j % 2's: its scores are issued two tiles ahead, behind the products that read the weights they overwrite.
          // There is one job, so items are numbered from 0.
          const auto slot_of = [&](int item) { return static_cast<uint32_t>(item) % S::kHalfSlots; };
          const auto wait_of = [&](int item) { return full + 8 * slot_of(item); };
          const auto phase_of = [&](int item) { return static_cast<uint32_t>(item) / S::kHalfSlots & 1; };
          going = warp_wait(q_full, 0, &failed);
          for (int j = 0; j < 2 && j < n && going; j++) {
            going = warp_wait(wait_of(2 * j), phase_of(2 * j), &failed);
            if (going && elected()) {
              scores(j, slot_of(2 * j));
              products_done(empty + 8 * slot_of(2 * j));
            }
            __syncwarp();
          }
#pragma unroll 1
          for (int j = 0; j < n && going; j++) {
            const int u = j & 1;
            const bool more = j + 2 < n;
            going = warp_wait_all(p_full + 8 * u, j >> 1 & 1, wait_of(2 * j + 1), phase_of(2 * j + 1), more ? wait_of(2 * j + 4) : 0, phase_of(2 * j + 4), &failed);
            if (!going) break;
            tmem_after_sync();
            if (elected()) {
              const uint32_t o = tmem + o_column + 128 * u, values_at = values + slot_of(2 * j + 1) * (S::kTile >> 4);
              product_over_tokens(o, tmem + 128 * u, values_at, kResults, j >= 2);
              product_over_tokens(o, tmem + 128 * u + 64, values_at + kHalfTokens, kResults, true);
              products_done(empty + 8 * slot_of(2 * j + 1));
              if (more) {
                scores(u, slot_of(2 * j + 4));
                products_done(empty + 8 * slot_of(2 * j + 4));
              } else {
                products_done(o_full + 8 * u);
              }
            }
            __syncwarp();
          }
          break;
        }
        int last_of[2] = {n - 1, n - 1};                // each one's last tile of keys
#pragma unroll
        for (int u = 0; u < 2; u++) {
          while (last_of[u] >= 0 && !active(u, last_of[u])) last_of[u]--;
        }
        bool begun[2] = {false, false};
        going = warp_wait(full + 8 * k.slot, k.phase, &failed);
#pragma unroll
        for (int u = 0; u < 2; u++) {
          if (u >= users || !going) break;
          going = warp_wait(q_full + 8 * u, loaded[u]++ & 1, &failed);
          if (going && elected()) {
            if (active(u, 0)) scores(u, k.slot);
            // without another tile, or with none at all, the queries are no longer needed
            if (last_of[u] <= 0) products_done(q_empty + 8 * u);
            if (u + 1 == users) products_done(empty + 8 * k.slot);
          }
          __syncwarp();
        }
        if (!going) break;
        // The tensor cores run a product or two behind the thread that issues them, so between two groups of products there is one
        // look at barriers and no more: with the last group of a tile of keys, at those of the next one's tiles too.
        Ring<S::kSlots> v = k;
        v.next();
        k = v;
        k.next();
        going = warp_wait_all(full + 8 * v.slot, v.phase, n > 1 ? full + 8 * k.slot : 0, k.phase, 0, 0, &failed);
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
                product_over_tokens(o, tmem + 128 * u, values_at, kResults, begun[u]);
                product_over_tokens(o, tmem + 128 * u + 64, values_at + kHalfTokens, kResults, true);
                if (j == last_of[u]) products_done(o_full + 8 * u);
              }
              if (last) products_done(empty + 8 * v.slot);
              // products run in the order in which they are issued: these scores overwrite P after it has been read
              if (more) scores(u, k.slot);
              if (j + 1 == last_of[u]) products_done(q_empty + 8 * u);
              if (last && j + 1 < n) products_done(empty + 8 * k.slot);
            }
            __syncwarp();
            done[u] += weighs;
            begun[u] = begun[u] || weighs;
          }
          if (j + 1 < n) {
            v = next_v;
            k = next_k;
          }
        }
        // k is the key item of a tile behind the last: the next job's first
      }
      if (!going) products_end(ended);
    } else if (warp == 19) {
      // -------------------------------------------------- masks: which keys are read, and zeros where values are not
      uint32_t r = 0, item = 1;                         // partial tiles; values in the ring
      bool going = true;
      for (int id = blockIdx.x; id < jobs && going; id += gridDim.x) {
        const Work w = work_of<kPaged>(f, id, first_place);
        for (int j = 0; j < w.n && going; j++, item += 2) {
          if (!gaps && w.template whole<kPaged>(j, p.tokens)) continue;
          uint32_t words[4];
          for (int i = 0; i < 4; i++) {
            const int key = w.tile(j) * 128 + i * 32 + lane;
            bool read = kPaged ? key < w.all.sinks || (key >= w.all.from && key < w.all.to) : key < w.seq.end;
            if (gaps && read) read = page_of(p.cache, w.job.batch, key) >= 0;
            words[i] = __ballot_sync(~0u, read);
          }
          // the next such tile may be at the end of the last job
          going = warp_wait_behind(landed + 8 * (r % kMaskRing), r / kMaskRing & 1, &failed, &progress);
          if (!going) break;
          const uint32_t values = ring_at + item % slots * S::kTile;
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
            barrier_arrive(full + 8 * (item % slots));
            barrier_arrive(masked + 8 * (r % kMaskRing));
          }
          r++;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------------------------------------------- softmax: a row belongs to two threads, one for each half of the keys of a tile
    // A wait that ran out does not end a job: the two warps of a row's threads meet at a barrier for every tile.
    const uint32_t lanes = static_cast<uint32_t>(32 * part) << 16;
    const uint32_t scores_at = tmem + 128 * t + 64 * half + lanes, result = tmem + o_column + 128 * t + half * (kDim / 2) + lanes;
    const float c = p.scale * kLog2e;
    uint32_t done = 0, ends = 0;       // tiles of keys and jobs of this tile of rows
    volatile int* const stop = &gave_up[t][part];
    for (int id = blockIdx.x; id < jobs; id += gridDim.x) {
      const Work w = work_of<kPaged>(f, id, first_place);
      if (!f.halves && t >= w.row_tiles) continue;
      const int token = w.job.q0 + row_token, in_group = w.job.chunk * tile_heads + row_head;
      const bool there = row < tile_heads * tile_tokens && token < p.tokens && in_group < p.group;   // the row is in the result
      const bool reads = there && token < w.seq.fresh;
      const bool tree = kPaged && p.tree;
      Reach mine = {0, 0, 0};
      if (reads) mine = tree ? reach_of(p, w.seq, tree_place, min(w.seq.held, w.seq.end)) : reach_of(p, w.seq, w.seq.held + token, min(w.seq.held + token + 1, w.seq.end));
      const Reach tile_reach = t ? w.of[1] : w.of[0];
      float top = -INFINITY, total = 0;
      bool begun = false;
#pragma unroll 1
      for (int j = 0; j < w.n; j++) {
        if (f.halves ? (j & 1) != t : !w.touches(tile_reach, j)) continue;
        uint32_t s[64];
        warp_wait(s_full + 8 * t, done & 1, &failed);
        tmem_after_sync();
        load_scores(scores_at, s);
        const int first_key = w.tile(j) * 128 + 64 * half;
        const bool whole_tile = (first_key >= mine.from && first_key + 64 <= mine.to) || first_key + 64 <= mine.sinks;
        if (!__all_sync(~0u, whole_tile) || gaps) {
          uint64_t read = bits_of(first_key, mine.from, mine.to) | bits_of(first_key, 0, mine.sinks);
          if (tree && reads) {
            const uint8_t* of_row = p.tree + w.job.batch * p.tree_batch + token * p.tree_token;
            for (int k = max(first_key, w.seq.held); k < min(first_key + 64, w.seq.end); k++) {
              if (of_row[k - w.seq.held]) read |= uint64_t{1} << (k - first_key);
            }
          }
          if (gaps) {
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
        if (!begun) {
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
        begun = true;
      }
      if (begun && !warp_wait(o_full + 8 * t, ends++ & 1, &failed)) *stop = 1;
      exchange[t][half][row] = total;
      asm volatile("bar.sync %0, 64;" : : "r"(1 + 4 * t + part) : "memory");
      total += exchange[t][half ^ 1][row];
      const bool stops = *stop;        // both warps of a row's threads end here, or neither
      asm volatile("bar.sync %0, 64;" : : "r"(1 + 4 * t + part) : "memory");   // the next job writes there
      if (stops) break;
      tmem_after_sync();
      // only a sum of 0 is a row without keys; one that is not a number stays so, in lse too
      const float by = total == 0 ? 0.0f : 1.0f / total;
      const float lse = total == 0 ? -INFINITY : top * p.scale + logf(total);
      const int64_t stat = (static_cast<int64_t>(w.job.batch) * p.q_heads + w.job.kv_head * p.group + in_group) * p.tokens + token;
      const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.tokens, slot = f.halves ? 2 * w.job.split + t : w.job.split;
#pragma unroll
      for (int x = 0; x < kDim / 2; x += 32) {
        uint32_t o[32] = {};
        if (begun) {
          tmem_load<32>(result + x, o);
          tmem_loaded(o);
        }
        if (f.parts > 1) {
          if (there && total != 0) {   // a part without keys is not read when they are joined
            float* to = f.part_out + (slot * rows + stat) * p.head_dim + half * (kDim / 2) + x;
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 8; i++) v[i] = __float_as_uint(__uint_as_float(o[k + i]) * by);
              if (half * (kDim / 2) + x + k < p.head_dim) store_row_part(to + k, v, 2);   // eight floats, as long as two units of elements
            }
          }
          continue;
        }
        T* const to = reinterpret_cast<T*>(p.out.data) + w.job.batch * p.out.batch + token * p.out.token + (w.job.kv_head * p.group + in_group) * p.out.head;
#pragma unroll
        for (int k = 0; k < 32; k += 16) {
          uint32_t v[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            // what a row without keys has summed is nothing, whatever stands there
            v[i] = total != 0 ? pack2<T>(__uint_as_float(o[k + 2 * i]) * by, __uint_as_float(o[k + 2 * i + 1]) * by) : 0u;
          }
          const int column = half * (kDim / 2) + x + k;
          if (there) store_row_part(to + column, v, (p.head_dim - column) / 8);
        }
      }
      if (half == 0 && there) {
        if (f.parts > 1) f.part_lse[slot * rows + stat] = lse;
        else if (p.lse) p.lse[stat] = lse;
      }
    }
  }
  __syncwarp();
  tmem_before_sync();
  __syncthreads();
  if (warp == 17) tmem_free<512>(tmem);
  if (failed) {   // not a number, instead of whatever the memory held, in all that the CTA was to write
    for (int id = block_again(); id < jobs; id += gridDim.x) {
      const Job at = job_of(f, id);
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
  int sms = 0;
  if (device_sms(p.device, &sms) != MLXD_OK) return cudaErrorInvalidDevice;
  const int64_t jobs = jobs_of(f);
  return launch_behind(causal_forward_kernel<T, kDim, kPaged>, dim3(static_cast<unsigned>(kPaged ? jobs : std::min<int64_t>(jobs, sms))), kThreads, bytes, stream, 1, f, maps);
}

template <class T>
cudaError_t launch_join(const ForwardParams& f, cudaStream_t stream) {
  const CausalParams& p = f.p;
  return launch_behind(causal_join_kernel<T>, dim3(static_cast<unsigned>((static_cast<int64_t>(p.batch) * p.q_heads * p.tokens + kJoinWarps - 1) / kJoinWarps)),
                       32 * kJoinWarps, 0, stream, 1, f);
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
  // Samples and splits lie along the grid's third dimension, up to 64 splits each; more samples go by tiles of 128 rows, of which a single
  // token leaves most empty (8 heads on 2 of 128, up to 1501 keys: 1023 samples 204 us, 1024 381; up to 101 keys 30 and 148).
  f.steps = paged && sixteens <= 1 && p.kv_heads <= 65535 && p.batch * int64_t{64} <= 65535;
  f.halves = paged && !f.steps && f.rows.tiles == 1;
  if (f.steps) {
    int64_t reach = p.cache.capacity;
    if (p.window != INT32_MAX) reach = std::min(reach, static_cast<int64_t>(p.window) + p.tokens + std::min(p.sinks, p.cache.capacity) + 32);
    // A CTA for each SM at most, joined within clusters of up to eight, where that leaves it 800 keys or fewer.  Else shares of a key head's
    // keys: up to 320 CTAs in all, of 128 keys at least, dealt to clusters; long stretches are cut at 1500 keys and by splits alone,
    // since samples are of different lengths and clusters wait for places side by side.  us for clusters x splits, what this takes first:
    // 8 heads, 1602 keys 8x1 8.0, 8x2 14.7, 4x4 9.8; 32 heads, 1505 keys 4x1 7.9, 8x1 10.6; 3001 keys 4x1 14.8, 8x1 18.7; 128 heads, up to
    // 24001 keys 1x16 220, 1x1 276, 2x1 371, 8x2 238.  Not the best everywhere: 8 heads, 6001 keys 8x1 15.0, 8x4 13.7, 4x4 13.3; 24001 keys
    // 8x5 30.6, 8x1 41.7, 8x4 27.9, 4x4 27.5; 160 heads, windows of 1028 keys 2x1 18.7, 1x1 28.7, 4x1 20.3, 1x2 17.3.
    while (f.cluster < 8 && 2 * heads * f.cluster <= sms && f.cluster * 2 <= reach / 128) f.cluster *= 2;
    if (heads * f.cluster > sms || reach > 800 * f.cluster) {
      f.cluster = 1;
      const int64_t shares = std::max<int64_t>(1, std::min(320 / heads, reach / 128));
      if (reach / shares > 1500) {
        const int64_t slots = static_cast<int64_t>(step_ctas(p.head_dim, p.tokens * p.group <= 8 ? 1 : 2)) * sms;
        f.splits = static_cast<int>(std::max(shares, std::min({reach / 1500, 8 * slots / heads, int64_t{64}})));
      } else {
        while (f.cluster < 8 && f.cluster * 2 <= shares) f.cluster *= 2;
        f.splits = static_cast<int>(shares / f.cluster);
      }
    }
    f.parts = f.splits;
    return f;
  }
  const int64_t ctas = static_cast<int64_t>((f.rows.tiles + (f.halves ? 0 : 1)) / (f.halves ? 1 : 2)) * f.rows.chunks * p.batch * p.kv_heads;
  if (paged) {
    // tiles of keys that a CTA may have
    int64_t most = (p.cache.capacity + 127) / 128;
    if (p.window != INT32_MAX) most = std::min(most, (static_cast<int64_t>(p.window) + 2 * f.rows.tokens + 127) / 128 + 1 + (std::min(p.sinks, p.cache.capacity) + 127) / 128);
    f.splits = static_cast<int>(std::max<int64_t>(1, std::min(most, std::min<int64_t>(sms / ctas, 64))));
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
