// Cached attention of few rows - single tokens of a generation, short drafts - where reading keys and values is all the work.
//
// A CTA takes up to 16 rows (tokens and the query heads that share a key head) and a stretch of the keys; its warps take 16 keys each
// in turn, as operands of 16 x 8 x 16 products.  Which elements of a head a product sums over, and which become its columns, is a
// matter of naming, so what a lane copies in units of 16 bytes is its own operands: copies go into a queue in shared memory that every lane
// has for itself, two to four rounds deep, and nothing waits for another lane.  Keys that are not read, or have no page, arrive as zeros.  The
// CTAs of a cluster share a stretch of keys and join their sums through each other's shared memory; where that is not enough CTAs, keys are
// split among clusters too, and a second kernel joins the parts.
//
// Reading keys and values once is the floor.  Measured: 32 heads on 8 of 128, 1602 keys: 8.0 us (17 keys 5.2: launch, lengths, pages,
// keys, one after another); sixteen sequences of up to 24001 keys 222-232 us, 4.8 TB/s (74 % of the measured rate), wherever pages lie and
// however long they are; forty sequences, windows of 1024, 16 heads on 4 of 64: 19 us.  Copies of 16 bytes keep half of the cycles of L1
// busy; beginnings and ends of CTAs take the rest.
#include "causal.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kKeys = 16;              // of a warp at a time
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;         // as in the kernel for many queries

template <class T> __device__ void product16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void product16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void product16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes to shared memory, zeros where nothing is there.
__device__ __forceinline__ void copy_unit(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" : : "r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint4 shared_unit(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Every thread of the cluster's CTAs: what they wrote to shared memory before is seen behind it.
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" : : : "memory");
}

__device__ __forceinline__ uint32_t of_rank(uint32_t at, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}

__device__ __forceinline__ float remote_float(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ float4 remote_float4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// kAlone: no more CTAs than SMs, so one CTA of an SM has twice the warps: a round of a warp takes 1 to 2 us, most of it one instruction
// waiting for another, and only other warps fill that.
template <int kDim, int kBlocks, bool kAlone>
struct StepSizes {
  static constexpr int kWarps = kAlone ? 8 : 4;
  static constexpr int kUnits = kDim / 32;         // 16-byte units of a key that a lane holds
  static constexpr int kHalves = kDim / 64;        // and of a value
  static constexpr int kCtas = kAlone ? 1 : step_ctas(kDim, kBlocks);   // of an SM, by registers
  static constexpr int kStages = kAlone ? 256 / kDim : (kDim == 128 ? 6 : 12) / kCtas;
  static_assert(2 * kStages <= 32, "two bits of a word for each");   // `holes`
  static constexpr int kStage = (2 * kUnits + 4 * kHalves) * 512;   // bytes of a warp's 16 keys and values
  static constexpr int kQueue = kWarps * kStages * kStage;
  // after the keys, in the same place: the warps' sums, then the CTA's
  static constexpr int kStride = kDim + 4;
  static constexpr int kSums = (kWarps + 1) * 8 * kBlocks * kStride * 4;
  static constexpr int kShared = kQueue > kSums ? kQueue : kSums;
};

// kBlocks: columns of eight rows.  Scores lie keys by rows, S^T = K Q^T, and results elements by rows, O^T = V^T P^T, so that eight rows (a token
// of up to eight heads) cost half of what sixteen do.
template <class T, int kDim, int kBlocks, bool kAlone>
__global__ void __launch_bounds__(32 * StepSizes<kDim, kBlocks, kAlone>::kWarps, StepSizes<kDim, kBlocks, kAlone>::kCtas)
    causal_step_kernel(const __grid_constant__ ForwardParams f) {
  using Z = StepSizes<kDim, kBlocks, kAlone>;
  constexpr int kWarps = Z::kWarps, kUnits = Z::kUnits, kHalves = Z::kHalves, kRows = 8 * kBlocks;
  const CausalParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ Reach reaches[kRows];
  __shared__ float warp_top[kWarps][kRows], warp_total[kWarps][kRows], cta_top[kRows], cta_total[kRows];
  asm volatile("griddepcontrol.launch_dependents;");
  wait_for_kernels_before();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, c = lane & 3;
  // neighbours are the key heads of the same keys, which lie side by side in a page
  const int kv_head = blockIdx.y, split = blockIdx.z % f.splits, batch = blockIdx.z / f.splits, rows = p.tokens * p.group;
  const Sequence seq = sequence_of<true>(p, batch);

  uint32_t q[kBlocks][kUnits][4];      // rows g, 8 + g; lane (g, c) holds the units c, c + 4, ...
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    const int row = 8 * b + g, token = row / p.group;
    const T* from = reinterpret_cast<const T*>(p.q.data) + batch * p.q.batch + token * p.q.token + (kv_head * p.group + row % p.group) * p.q.head;
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const uint4 x = row < rows && 32 * i + 8 * c < p.head_dim ? *reinterpret_cast<const uint4*>(from + 32 * i + 8 * c) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < 4; w++) q[b][i][w] = word_of(x, w);
    }
  }

  // ---------------------------------------------------- what each row reads: eight threads a row
  if (threadIdx.x < 8 * kRows) {
    const int row = threadIdx.x / 8, token = row / p.group;
    const bool reads = row < rows && token < seq.fresh;
    int place = seq.held + token, to = min(place + 1, seq.end);
    if (p.tree) {
      const uint8_t* tree = p.tree + batch * p.tree_batch + token * p.tree_token;
      int others = 0;
      for (int j = threadIdx.x % 8; reads && j < seq.fresh; j += 8) others += j != token && tree[j];
      for (int d = 4; d; d >>= 1) others += __shfl_xor_sync(~0u, others, d);
      place = seq.held + others;
      to = min(seq.held, seq.end);
    }
    if (threadIdx.x % 8 == 0) reaches[row] = reads ? reach_of(p, seq, place, to) : Reach{-1, 0, 0};
  }
  __syncthreads();
  // of all rows: what some row reads, and what every row reads
  Reach all, every;
  {
    const Reach r = reaches[lane % kRows];
    const bool reads = r.sinks >= 0;
    all.sinks = __reduce_max_sync(~0u, reads ? r.sinks : 0);
    all.from = __reduce_min_sync(~0u, reads ? r.from : INT32_MAX);
    all.to = __reduce_max_sync(~0u, reads ? r.to : 0);
    every.sinks = __reduce_min_sync(~0u, reads ? r.sinks : INT32_MAX);
    every.from = __reduce_max_sync(~0u, reads ? r.from : 0);
    every.to = __reduce_min_sync(~0u, reads ? r.to : INT32_MAX);
    if (__any_sync(~0u, reads) && p.tree) {   // the new tokens are read by the tree alone
      all.from = min(all.from, min(seq.held, seq.end));
      all.to = seq.end;
    }
    all.from = min(all.from, all.to);
    all.sinks = min(all.sinks, all.from);
  }
  // the list of sixteens of keys: first ones, then the window's
  const int sink_list = (all.sinks + kKeys - 1) / kKeys, main_first = max(all.from / kKeys, sink_list);
  const int whole = sink_list + (all.to > all.from ? max((all.to + kKeys - 1) / kKeys - main_first, 0) : 0);
  const int shares = f.splits * f.cluster, share = (whole + shares - 1) / shares;
  const int first = min((split * f.cluster + static_cast<int>(blockIdx.x)) * share, whole), n = min(share, whole - first);
  const auto key_of = [&](int j) { return (j + first < sink_list ? j + first : j + first - sink_list + main_first) * kKeys; };

  // ---------------------------------------------------- copies
  // Pages of this warp's next sixteen rounds, two a round (a page has at least eight keys): a lane each, loaded sixteen rounds ahead.
  const auto pages_from = [&](int j) {
    const int mine = j + (lane >> 1) * kWarps;
    return mine < n ? page_of(p.cache, batch, key_of(mine) + 8 * (lane & 1)) : -1;
  };
  const uint32_t queue = smem_address(shared) + warp * Z::kStages * Z::kStage + lane * 16;
  // lane (g, c) takes of the keys g and 8 + g the units c, c + 4, ..., of the values 2 c, 2 c + 1, 2 c + 8, 2 c + 9 the units g, g + 8
  const T* const key_pool = reinterpret_cast<const T*>(p.k.data) + kv_head * p.k.head + g * p.k.token + 8 * c;
  const T* const value_pool = reinterpret_cast<const T*>(p.v.data) + kv_head * p.v.head + 2 * c * p.v.token + 8 * g;
  int pages = pages_from(warp), next_pages = pages_from(warp + 16 * kWarps), copied = warp, round = 0;
  uint32_t holes = 0;                  // two bits a stage: halves without a page
  const auto copy = [&](int stage) {   // round `copied` of this warp, which may be none
    const int here = round & 15;
    const int page0 = __shfl_sync(~0u, pages, 2 * here), page1 = __shfl_sync(~0u, pages, 2 * here + 1);
    if (copied < n) {
      const int at = key_of(copied), row0 = at & (p.cache.page_size - 1), row1 = (at + 8) & (p.cache.page_size - 1);
      const uint32_t to = queue + stage * Z::kStage;
      const bool inside = (at >= all.from && at + kKeys <= all.to) || at + kKeys <= all.sinks;   // every key is read by some row
      const auto read = [&](int key) { return inside || key < all.sinks || (key >= all.from && key < all.to); };
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int page = h ? page1 : page0, row = h ? row1 : row0;
        const T* const keys = key_pool + max(page, 0) * p.k.batch + row * p.k.token;
        const T* const values = value_pool + max(page, 0) * p.v.batch + row * p.v.token;
        const bool there = page >= 0 && read(at + 8 * h + g);
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
          const bool whole = there && 32 * i + 8 * c < p.head_dim;
          copy_unit(to + (h * kUnits + i) * 512, whole ? keys + 32 * i : key_pool, whole);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const bool there = page >= 0 && read(at + 8 * h + 2 * c + e);
#pragma unroll
          for (int i = 0; i < kHalves; i++) {
            const bool whole = there && 64 * i + 8 * g < p.head_dim;
            copy_unit(to + (2 * kUnits + (2 * h + e) * kHalves + i) * 512, whole ? values + e * p.v.token + 64 * i : value_pool, whole);
          }
        }
      }
      holes = (holes & ~(3u << (2 * stage))) | (static_cast<uint32_t>((page0 < 0) | (page1 < 0) << 1) << (2 * stage));
    }
    asm volatile("cp.async.commit_group;" : : : "memory");
    copied += kWarps;
    if ((++round & 15) == 0) {
      pages = next_pages;
      next_pages = pages_from(copied + 16 * kWarps);
    }
  };
#pragma unroll
  for (int i = 0; i < Z::kStages; i++) copy(i);

  const float scale = p.scale * kLog2e;
  float top[kBlocks][2], total[kBlocks][2] = {};   // of rows 2 c, 2 c + 1 (and 8 more)
#pragma unroll
  for (int b = 0; b < kBlocks; b++) top[b][0] = top[b][1] = -INFINITY;
  constexpr int kProducts = kDim / 16;
  float o[kBlocks][kProducts][4] = {};
  int stage = 0;
  for (int j = warp; j < n; j += kWarps) {
    asm volatile("cp.async.wait_group %0;" : : "n"(Z::kStages - 1) : "memory");
    const uint32_t from = queue + stage * Z::kStage;
    float s[kBlocks][4] = {}, s2[kBlocks][4] = {};   // keys g (values 0, 1) and 8 + g (2, 3) of rows 2 c, 2 c + 1
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const uint4 k0 = shared_unit(from + i * 512), k1 = shared_unit(from + (kUnits + i) * 512);
      const uint32_t a[4] = {k0.x, k1.x, k0.y, k1.y}, b[4] = {k0.z, k1.z, k0.w, k1.w};
#pragma unroll
      for (int x = 0; x < kBlocks; x++) {
        product16<T>(s[x], a, q[x][i][0], q[x][i][1]);
        product16<T>(s2[x], b, q[x][i][2], q[x][i][3]);
      }
    }
#pragma unroll
    for (int x = 0; x < kBlocks; x++) {
#pragma unroll
      for (int e = 0; e < 4; e++) s[x][e] += s2[x][e];
    }
    const int at = key_of(j);
    const uint32_t missing = holes >> (2 * stage) & 3;
    if (missing || !((at >= every.from && at + kKeys <= every.to) || at + kKeys <= every.sinks)) {
#pragma unroll
      for (int x = 0; x < kBlocks; x++) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int row = 8 * x + 2 * c + r;
          const Reach reach = reaches[row];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int key = at + 8 * h + g;
            bool read = key < reach.sinks || (key >= reach.from && key < reach.to);
            if (p.tree && reach.sinks >= 0 && key >= seq.held && key < seq.end) read = p.tree[batch * p.tree_batch + row / p.group * p.tree_token + key - seq.held];
            if (!read || (missing >> h & 1)) s[x][2 * h + r] = -INFINITY;
          }
        }
      }
    }
    // a row's reference is moved where some lane's score has grown by more than 2^8 in weight
    float now[kBlocks][2];
    bool grows = false;
#pragma unroll
    for (int x = 0; x < kBlocks; x++) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        now[x][r] = fmaxf(s[x][r], s[x][2 + r]);
        grows = grows || (now[x][r] - top[x][r]) * scale > kSlack;
      }
    }
    if (__any_sync(~0u, grows)) {
#pragma unroll
      for (int x = 0; x < kBlocks; x++) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float most = now[x][r];
          for (int d = 4; d < 32; d *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
          const bool moves = (most - top[x][r]) * scale > kSlack;   // also from -infinity; not where both are
          const float keep = moves ? exp2_of((top[x][r] - most) * scale) : 1.0f;
          top[x][r] = moves ? most : top[x][r];
          total[x][r] *= keep;
#pragma unroll
          for (int i = 0; i < kProducts; i++) {
            o[x][i][r] *= keep;
            o[x][i][2 + r] *= keep;
          }
        }
      }
    }
    uint32_t w[kBlocks][2];
#pragma unroll
    for (int x = 0; x < kBlocks; x++) {
      const float base[2] = {top[x][0] == -INFINITY ? 0.0f : -top[x][0] * scale, top[x][1] == -INFINITY ? 0.0f : -top[x][1] * scale};
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float y = exp2_of(fmaf(s[x][2 * h], scale, base[0])), z = exp2_of(fmaf(s[x][2 * h + 1], scale, base[1]));
        total[x][0] += y;
        total[x][1] += z;
        // an operand of the products, so 16 bits (the sum is of the floats), keys by rows to rows by keys
        const uint32_t packed = pack2<T>(y, z);
        asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w[x][h]) : "r"(packed));
      }
    }
    uint4 v[4][kHalves];
#pragma unroll
    for (int h = 0; h < 4; h++) {
#pragma unroll
      for (int i = 0; i < kHalves; i++) v[h][i] = shared_unit(from + (2 * kUnits + h * kHalves + i) * 512);
    }
    // Heads of 128: rows g and 8 + g of product i are the elements 8 g + i and 64 + 8 g + i; of 64: 8 g + 2 i and 8 g + 2 i + 1.
#pragma unroll
    for (int i = 0; i < kProducts; i++) {
      const int e0 = kHalves == 2 ? i : 2 * i, e1 = kHalves == 2 ? i : 2 * i + 1;
      const auto pair = [&](int h, int half, int e) { return __byte_perm(word_of(v[h][half], e / 2), word_of(v[h + 1][half], e / 2), e & 1 ? 0x7632 : 0x5410); };
      const uint32_t a[4] = {pair(0, 0, e0), pair(0, kHalves - 1, e1), pair(2, 0, e0), pair(2, kHalves - 1, e1)};
#pragma unroll
      for (int x = 0; x < kBlocks; x++) product16<T>(o[x][i], a, w[x][0], w[x][1]);
    }
    copy(stage);
    stage = stage + 1 == Z::kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" : : : "memory");
  __syncthreads();                     // the queues are no longer needed

  // ---------------------------------------------------- the warps' sums together
  float* const warp_out = reinterpret_cast<float*>(shared);
  float* const cta_out = warp_out + kWarps * kRows * Z::kStride;
#pragma unroll
  for (int x = 0; x < kBlocks; x++) {
#pragma unroll
    for (int r = 0; r < 2; r++) {
      for (int d = 4; d < 32; d *= 2) total[x][r] += __shfl_xor_sync(~0u, total[x][r], d);
      const int row = 8 * x + 2 * c + r;
      if (g == 0) {
        warp_top[warp][row] = top[x][r];
        warp_total[warp][row] = total[x][r];
      }
      float* to = warp_out + (warp * kRows + row) * Z::kStride + 8 * g;
      if constexpr (kHalves == 2) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          *reinterpret_cast<float4*>(to + 64 * e) = make_float4(o[x][0][2 * e + r], o[x][1][2 * e + r], o[x][2][2 * e + r], o[x][3][2 * e + r]);
          *reinterpret_cast<float4*>(to + 64 * e + 4) = make_float4(o[x][4][2 * e + r], o[x][5][2 * e + r], o[x][6][2 * e + r], o[x][7][2 * e + r]);
        }
      } else {
        *reinterpret_cast<float4*>(to) = make_float4(o[x][0][r], o[x][0][2 + r], o[x][1][r], o[x][1][2 + r]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(o[x][2][r], o[x][2][2 + r], o[x][3][r], o[x][3][2 + r]);
      }
    }
  }
  __syncthreads();
  constexpr int kLanes = kDim / 4;     // threads of a row, 4 elements each
  for (int i = threadIdx.x; i < rows * kLanes; i += 32 * kWarps) {
    const int r = i / kLanes, x = i % kLanes * 4;
    float most = warp_top[0][r], sum = 0;
#pragma unroll
    for (int w = 1; w < kWarps; w++) most = fmaxf(most, warp_top[w][r]);
    const float base = most == -INFINITY ? 0.0f : most;
    float4 e = {};
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float by = exp2_of((warp_top[w][r] - base) * scale);
      const float4 a = *reinterpret_cast<const float4*>(warp_out + (w * kRows + r) * Z::kStride + x);
      sum += warp_total[w][r] * by;
      e.x += a.x * by;
      e.y += a.y * by;
      e.z += a.z * by;
      e.w += a.w * by;
    }
    *reinterpret_cast<float4*>(cta_out + r * Z::kStride + x) = e;
    if (x == 0) {   // a row that reads nothing has neither, whatever its scores were: tiles that every other row reads are not masked for it
      const bool reads = reaches[r].sinks >= 0;
      cta_top[r] = reads ? most : -INFINITY;
      cta_total[r] = reads ? sum : 0.0f;
    }
  }

  // ---------------------------------------------------- and the CTAs' of the cluster, each some of the rows' elements
  if (f.cluster > 1) cluster_meet();
  else __syncthreads();
  const uint32_t rank = f.cluster > 1 ? cluster_rank() : 0;
  const uint32_t out_at = smem_address(cta_out), top_at = smem_address(cta_top), total_at = smem_address(cta_total);
  for (int i = rank * 32 * kWarps + threadIdx.x; i < rows * kLanes; i += 32 * kWarps * f.cluster) {
    const int r = i / kLanes, x = i % kLanes * 4, token = r / p.group, head = kv_head * p.group + r % p.group;
    float most = -INFINITY, sum = 0;
    for (int k = 0; k < f.cluster; k++) most = fmaxf(most, remote_float(of_rank(top_at + 4 * r, k)));
    const float base = most == -INFINITY ? 0.0f : most;
    float4 e = {};
    for (int k = 0; k < f.cluster; k++) {
      const float by = exp2_of((remote_float(of_rank(top_at + 4 * r, k)) - base) * scale);
      const float4 a = remote_float4(of_rank(out_at + (r * Z::kStride + x) * 4, k));
      sum += remote_float(of_rank(total_at + 4 * r, k)) * by;
      e.x += a.x * by;
      e.y += a.y * by;
      e.z += a.z * by;
      e.w += a.w * by;
    }
    if (x >= p.head_dim) continue;
    // only a sum of 0 is a row without keys; one that is not a number stays so, in lse too, where the joining finds it
    const float by = 1.0f / sum;
    if (sum == 0) e = make_float4(0, 0, 0, 0);
    else e = make_float4(e.x * by, e.y * by, e.z * by, e.w * by);
    const float lse = sum == 0 ? -INFINITY : most * p.scale + logf(sum);
    const int64_t stat = (static_cast<int64_t>(batch) * p.q_heads + head) * p.tokens + token;
    if (f.splits > 1) {
      const int64_t part = split * static_cast<int64_t>(p.batch) * p.q_heads * p.tokens + stat;
      *reinterpret_cast<float4*>(f.part_out + part * p.head_dim + x) = e;
      if (x == 0) f.part_lse[part] = lse;
    } else {
      T* to = reinterpret_cast<T*>(p.out.data) + batch * p.out.batch + token * p.out.token + head * p.out.head + x;
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(e.x, e.y), pack2<T>(e.z, e.w));
      if (x == 0 && p.lse) p.lse[stat] = lse;
    }
  }
  if (f.cluster > 1) cluster_meet();   // nobody leaves while others read what it has
}

template <class T, int kDim, int kBlocks, bool kAlone>
cudaError_t launch(const ForwardParams& f, cudaStream_t stream) {
  constexpr int bytes = StepSizes<kDim, kBlocks, kAlone>::kShared;
  const CausalParams& p = f.p;
  const cudaError_t e = allow_shared<causal_step_kernel<T, kDim, kBlocks, kAlone>>(bytes, p.device);
  if (e != cudaSuccess) return e;
  return launch_behind(causal_step_kernel<T, kDim, kBlocks, kAlone>, dim3(f.cluster, p.kv_heads, f.splits * p.batch), 32 * StepSizes<kDim, kBlocks, kAlone>::kWarps, bytes, stream, f.cluster, f);
}

template <class T, int kDim, int kBlocks>
cudaError_t launch(const ForwardParams& f, cudaStream_t stream) {
  int sms = 0;
  if (device_sms(f.p.device, &sms) != MLXD_OK) return cudaErrorInvalidDevice;
  const int64_t ctas = static_cast<int64_t>(f.cluster) * f.splits * f.p.batch * f.p.kv_heads;
  return ctas <= sms ? launch<T, kDim, kBlocks, true>(f, stream) : launch<T, kDim, kBlocks, false>(f, stream);
}

template <class T>
cudaError_t launch(const ForwardParams& f, cudaStream_t stream) {
  if (f.p.tokens * f.p.group <= 8) return f.p.head_dim > 64 ? launch<T, 128, 1>(f, stream) : launch<T, 64, 1>(f, stream);
  return f.p.head_dim > 64 ? launch<T, 128, 2>(f, stream) : launch<T, 64, 2>(f, stream);
}

}  // namespace

cudaError_t launch_causal_step(const ForwardParams& f, int dtype, cudaStream_t stream) {
  return dtype == MLXD_F16 ? launch<__half>(f, stream) : launch<__nv_bfloat16>(f, stream);
}

}  // namespace mlxd
