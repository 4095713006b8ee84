// Cached attention of few rows - single tokens of a generation, short drafts - where reading keys and values is all the work.
//
// A CTA takes up to 16 rows (tokens and the query heads that share a key head) and a stretch of the keys; its four warps take 16 keys each
// in turn, as operands of 16 x 8 x 16 products.  Which elements of a head a product sums over, and which become its columns, is a
// matter of naming, so what a lane copies in units of 16 bytes is its own operands: copies go into a queue in shared memory that every lane
// has for itself, three rounds deep, and nothing waits for another lane.  Keys that are not read, or have no page, arrive as zeros.  The
// CTAs of a cluster share a stretch of keys and join their sums through each other's shared memory; where that is not enough CTAs, keys are
// split among clusters too, and a second kernel joins the parts.
#include "causal.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kWarps = 4;
constexpr int kRows = 16;
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

template <int kDim>
struct StepSizes {
  static constexpr int kUnits = kDim / 32;         // 16-byte units of a key that a lane holds
  static constexpr int kHalves = kDim / 64;        // and of a value
  static constexpr int kStages = kDim == 128 ? 3 : 6;
  static constexpr int kStage = (2 * kUnits + 4 * kHalves) * 512;   // bytes of a warp's 16 keys and values
  static constexpr int kQueue = kWarps * kStages * kStage;
  // after the keys, in the same place: the warps' sums, then the CTA's
  static constexpr int kStride = kDim + 4;
  static constexpr int kWarpSums = kWarps * kRows * kStride * 4;
  static constexpr int kShared = kQueue > kWarpSums + kRows * kStride * 4 ? kQueue : kWarpSums + kRows * kStride * 4;
};

template <class T, int kDim>
__global__ void __launch_bounds__(32 * kWarps, 2) causal_step_kernel(const __grid_constant__ ForwardParams f) {
  using Z = StepSizes<kDim>;
  constexpr int kUnits = Z::kUnits, kHalves = Z::kHalves;
  const CausalParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t shared[];
  __shared__ Reach reaches[kRows];
  __shared__ float warp_top[kWarps][kRows], warp_total[kWarps][kRows], cta_top[kRows], cta_total[kRows];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, c = lane & 3;
  const int kv_head = blockIdx.y % p.kv_heads, batch = blockIdx.y / p.kv_heads, row0 = blockIdx.z * kRows, rows = p.tokens * p.group;
  const Sequence seq = sequence_of<true>(p, batch);

  uint32_t q[2][kUnits][4];            // rows g and 8 + g; lane (g, c) holds the units c, c + 4, ...
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int row = row0 + 8 * h + g, token = row / p.group;
    const T* from = reinterpret_cast<const T*>(p.q.data) + batch * p.q.batch + token * p.q.token + (kv_head * p.group + row % p.group) * p.q.head;
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const uint4 x = row < rows && 32 * i + 8 * c < p.head_dim ? __ldg(reinterpret_cast<const uint4*>(from + 32 * i + 8 * c)) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < 4; w++) q[h][i][w] = word_of(x, w);
    }
  }

  // ---------------------------------------------------- what each row reads: eight threads a row
  {
    const int row = row0 + threadIdx.x / 8, token = row / p.group;
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
    if (threadIdx.x % 8 == 0) reaches[threadIdx.x / 8] = reads ? reach_of(p, seq, place, to) : Reach{-1, 0, 0};
  }
  __syncthreads();
  // of all rows: what some row reads, and what every row reads
  Reach all = {0, INT32_MAX, 0}, every = {INT32_MAX, 0, INT32_MAX};
  const int mine = lane < kRows ? lane : 0;
  {
    const Reach r = reaches[mine];
    const bool reads = r.sinks >= 0;
    all.sinks = __reduce_max_sync(~0u, reads ? r.sinks : 0);
    all.from = __reduce_min_sync(~0u, reads ? r.from : INT32_MAX);
    all.to = __reduce_max_sync(~0u, reads ? r.to : 0);
    every.sinks = __reduce_min_sync(~0u, reads ? r.sinks : INT32_MAX);
    every.from = __reduce_max_sync(~0u, reads ? r.from : 0);
    every.to = __reduce_min_sync(~0u, reads ? r.to : INT32_MAX);
    const bool any = __any_sync(~0u, reads);
    if (any && p.tree) {               // the new tokens are read by the tree alone
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
  const int first = min(static_cast<int>(blockIdx.x) * share, whole), n = min(share, whole - first);
  const auto key_of = [&](int j) { return (j + first < sink_list ? j + first : j + first - sink_list + main_first) * kKeys; };

  // ---------------------------------------------------- copies
  // Pages of this warp's next sixteen rounds, two a round (a page has at least eight keys): a lane each, loaded sixteen rounds ahead.
  const auto pages_from = [&](int j) {
    const int mine = j + (lane >> 1) * kWarps;
    return mine < n ? page_of(p.cache, batch, key_of(mine) + 8 * (lane & 1)) : -1;
  };
  const uint32_t queue = smem_address(shared) + warp * Z::kStages * Z::kStage + lane * 16;
  const T* const key_pool = reinterpret_cast<const T*>(p.k.data) + kv_head * p.k.head;
  const T* const value_pool = reinterpret_cast<const T*>(p.v.data) + kv_head * p.v.head;
  int pages = pages_from(warp), next_pages = pages_from(warp + 16 * kWarps), copied = warp, round = 0;
  uint32_t holes = 0;                  // two bits a stage: halves without a page
  const auto copy = [&](int stage) {   // round `copied` of this warp, which may be none
    const int at = key_of(copied), here = round & 15;
    const int page0 = __shfl_sync(~0u, pages, 2 * here), page1 = __shfl_sync(~0u, pages, 2 * here + 1);
    if (copied < n) {
      const int row = at & (p.cache.page_size - 1), row1 = (at + 8) & (p.cache.page_size - 1);
      const uint32_t to = queue + stage * Z::kStage;
      const auto read = [&](int key) { return key < all.sinks || (key >= all.from && key < all.to); };
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int page = h ? page1 : page0;
        const T* from = key_pool + static_cast<int64_t>(max(page, 0)) * p.k.batch + ((h ? row1 : row) + g) * p.k.token + 8 * c;
        const bool there = page >= 0 && read(at + 8 * h + g);
#pragma unroll
        for (int i = 0; i < kUnits; i++) copy_unit(to + (h * kUnits + i) * 512, there && 32 * i + 8 * c < p.head_dim ? from + 32 * i : key_pool, there && 32 * i + 8 * c < p.head_dim);
      }
#pragma unroll
      for (int h = 0; h < 4; h++) {    // keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9; units g, g + 8
        const int page = h / 2 ? page1 : page0, key = 2 * c + (h & 1);
        const T* from = value_pool + static_cast<int64_t>(max(page, 0)) * p.v.batch + ((h / 2 ? row1 : row) + key) * p.v.token + 8 * g;
        const bool there = page >= 0 && read(at + 8 * (h / 2) + key);
#pragma unroll
        for (int i = 0; i < kHalves; i++) {
          copy_unit(to + (2 * kUnits + h * kHalves + i) * 512, there && 64 * i + 8 * g < p.head_dim ? from + 64 * i : value_pool, there && 64 * i + 8 * g < p.head_dim);
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
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {};
  float o[kHalves][8][4] = {};
  int stage = 0;
  for (int j = warp; j < n; j += kWarps) {
    asm volatile("cp.async.wait_group %0;" : : "n"(Z::kStages - 1) : "memory");
    const uint32_t from = queue + stage * Z::kStage;
    float s[2][4] = {};
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < kUnits; i++) {
        const uint4 k = shared_unit(from + (h * kUnits + i) * 512);
        const uint32_t a[4] = {q[0][i][0], q[1][i][0], q[0][i][1], q[1][i][1]}, b[4] = {q[0][i][2], q[1][i][2], q[0][i][3], q[1][i][3]};
        product16<T>(s[h], a, k.x, k.y);
        product16<T>(s[h], b, k.z, k.w);
      }
    }
    uint4 v[4][kHalves];
#pragma unroll
    for (int h = 0; h < 4; h++) {
#pragma unroll
      for (int i = 0; i < kHalves; i++) v[h][i] = shared_unit(from + (2 * kUnits + h * kHalves + i) * 512);
    }
    // a lane has rows g (values 0, 1) and 8 + g (2, 3) of keys 2 c, 2 c + 1 and 8 more
    const int at = key_of(j);
    const uint32_t missing = holes >> (2 * stage) & 3;
    if (missing || !((at >= every.from && at + kKeys <= every.to) || at + kKeys <= every.sinks)) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const Reach reach = reaches[8 * r + g];
        const int token = (row0 + 8 * r + g) / p.group;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int key = at + 8 * h + 2 * c + e;
            bool read = key < reach.sinks || (key >= reach.from && key < reach.to);
            if (p.tree && reach.sinks >= 0 && key >= seq.held && key < seq.end) read = p.tree[batch * p.tree_batch + token * p.tree_token + key - seq.held];
            if (!read || (missing >> h & 1)) s[h][2 * r + e] = -INFINITY;
          }
        }
      }
    }
    uint32_t w[4];
    float now[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      now[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      now[r] = fmaxf(now[r], __shfl_xor_sync(~0u, now[r], 1));
      now[r] = fmaxf(now[r], __shfl_xor_sync(~0u, now[r], 2));
    }
    const bool grows0 = (now[0] - top[0]) * scale > kSlack, grows1 = (now[1] - top[1]) * scale > kSlack;
    if (__any_sync(~0u, grows0 || grows1)) {
      const float keep[2] = {grows0 ? exp2_of((top[0] - now[0]) * scale) : 1.0f, grows1 ? exp2_of((top[1] - now[1]) * scale) : 1.0f};
      top[0] = grows0 ? now[0] : top[0];
      top[1] = grows1 ? now[1] : top[1];
      total[0] *= keep[0];
      total[1] *= keep[1];
#pragma unroll
      for (int x = 0; x < kHalves; x++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
          for (int e = 0; e < 4; e++) o[x][i][e] *= keep[e / 2];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const float base = top[r] == -INFINITY ? 0.0f : -top[r] * scale;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float x = exp2_of(fmaf(s[h][2 * r], scale, base)), y = exp2_of(fmaf(s[h][2 * r + 1], scale, base));
        total[r] += x + y;
        w[2 * h + r] = pack2<T>(x, y);   // an operand of the products, so 16 bits; the sum is of the floats
      }
    }
    // column n of product (x, i) is element 64 x + 8 n + i
#pragma unroll
    for (int x = 0; x < kHalves; x++) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int order = i & 1 ? 0x7632 : 0x5410;
        product16<T>(o[x][i], w, __byte_perm(word_of(v[0][x], i / 2), word_of(v[1][x], i / 2), order),
                     __byte_perm(word_of(v[2][x], i / 2), word_of(v[3][x], i / 2), order));
      }
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
  for (int r = 0; r < 2; r++) {
    total[r] += __shfl_xor_sync(~0u, total[r], 1);
    total[r] += __shfl_xor_sync(~0u, total[r], 2);
    if (c == 0) {
      warp_top[warp][8 * r + g] = top[r];
      warp_total[warp][8 * r + g] = total[r];
    }
#pragma unroll
    for (int x = 0; x < kHalves; x++) {
#pragma unroll
      for (int m = 0; m < 2; m++) {
        float* to = warp_out + (warp * kRows + 8 * r + g) * Z::kStride + 64 * x + 8 * (2 * c + m);
        *reinterpret_cast<float4*>(to) = make_float4(o[x][0][2 * r + m], o[x][1][2 * r + m], o[x][2][2 * r + m], o[x][3][2 * r + m]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(o[x][4][2 * r + m], o[x][5][2 * r + m], o[x][6][2 * r + m], o[x][7][2 * r + m]);
      }
    }
  }
  __syncthreads();
  constexpr int kLanes = kDim / 4;     // threads of a row, 4 elements each
  const int here = min(rows - row0, kRows);
  for (int i = threadIdx.x; i < here * kLanes; i += 32 * kWarps) {
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
    if (x == 0) {
      cta_top[r] = most;
      cta_total[r] = reaches[r].sinks < 0 ? 0.0f : sum;   // a row that reads nothing
    }
  }

  // ---------------------------------------------------- and the CTAs' of the cluster, each some of the rows' elements
  if (f.cluster > 1) cluster_meet();
  else __syncthreads();
  const uint32_t rank = f.cluster > 1 ? cluster_rank() : 0;
  const uint32_t out_at = smem_address(cta_out), top_at = smem_address(cta_top), total_at = smem_address(cta_total);
  for (int i = rank * 32 * kWarps + threadIdx.x; i < here * kLanes; i += 32 * kWarps * f.cluster) {
    const int r = i / kLanes, x = i % kLanes * 4, row = row0 + r, token = row / p.group, head = kv_head * p.group + row % p.group;
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
      const int64_t part = blockIdx.x / f.cluster * static_cast<int64_t>(p.batch) * p.q_heads * p.tokens + stat;
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

template <class T, int kDim>
cudaError_t launch(const ForwardParams& f, cudaStream_t stream) {
  constexpr int bytes = StepSizes<kDim>::kShared;
  const CausalParams& p = f.p;
  const cudaError_t e = allow_shared<causal_step_kernel<T, kDim>>(bytes, p.device);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(f.splits * f.cluster, p.batch * p.kv_heads, (static_cast<unsigned>(p.tokens) * p.group + kRows - 1) / kRows);
  config.blockDim = dim3(32 * kWarps);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = f.cluster;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = f.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&config, causal_step_kernel<T, kDim>, f);
}

}  // namespace

cudaError_t launch_causal_step(const ForwardParams& f, int dtype, cudaStream_t stream) {
  if (dtype == MLXD_F16) return f.p.head_dim > 64 ? launch<__half, 128>(f, stream) : launch<__half, 64>(f, stream);
  return f.p.head_dim > 64 ? launch<__nv_bfloat16, 128>(f, stream) : launch<__nv_bfloat16, 64>(f, stream);
}

}  // namespace mlxd
