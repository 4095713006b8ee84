// Cross attention of few queries - single tokens of a generation - where reading keys and values is all the work.
//
// A CTA takes up to 16 rows (tokens and heads that share a key head) and a stretch of the keys; its four warps take 16 keys each in
// turn, straight from memory into the registers of 16 x 8 x 16 products, with no detour through shared memory: which elements of a
// head a product sums over, and which become its columns, is a matter of naming, so a lane's 16-byte loads are its operands.
// Reading keys and values once is the floor.  Measured: 32 heads on 8, 1601 keys: 8.0 us with the joining of the parts; sixteen
// sequences of up to 6404 keys: 58 us, 4.7 TB/s (72 % of the measured rate): a CTA's first loads and its last sums are not hidden
// (two CTAs of 215 registers an SM).
#include "cross.h"
#include "sm100.cuh"

namespace mlxd {

namespace {

constexpr int kWarps = 4;
constexpr int kRows = 16;
constexpr int kKeys = 16;              // of a warp at a time
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;         // as in the kernel for many queries

struct StepParams {
  CrossParams p;
  int rows;                            // tokens * group
  int split_keys, splits;              // keys of a CTA; 1: results are final
  float* part_out;                     // [splits][batch, q_heads, q_tokens][head_dim]
  float* part_lse;                     // [splits][batch, q_heads, q_tokens]
};

template <class T> __device__ void product16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void product16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void product16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_unit(const void* at, bool there) {
  return there ? __ldg(static_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

template <class T, int kDim>
__global__ void __launch_bounds__(32 * kWarps, 2) cross_step_kernel(const __grid_constant__ StepParams sp) {
  const CrossParams& p = sp.p;
  constexpr int kUnits = kDim / 32;    // 16-byte units of a key that a lane holds
  __shared__ float warp_out[kWarps][kRows][kDim + 4];
  __shared__ float warp_top[kWarps][kRows], warp_total[kWarps][kRows];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, c = lane & 3;
  const int split = blockIdx.x, kv_head = blockIdx.y % p.kv_heads, batch = blockIdx.y / p.kv_heads, row0 = blockIdx.z * kRows;
  const int length = length_of(p, batch);
  const int first = split * sp.split_keys, end = min(length, first + sp.split_keys);
  if (first >= end && sp.splits > 1) return;   // the sum over the parts goes by the length too

  const T* keys = reinterpret_cast<const T*>(p.k.data) + batch * p.k.batch + kv_head * p.k.head;
  const T* values = reinterpret_cast<const T*>(p.v.data) + batch * p.v.batch + kv_head * p.v.head;
  const uint8_t* mask = p.key_mask ? p.key_mask + batch * p.key_mask_stride : nullptr;

  // lane (g, c) holds of key g, and of key 8 + g, the units c, c + 4, ...
  uint4 k[2][kUnits];
  const auto load_keys = [&](int from) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int key = from + 8 * h + g;
#pragma unroll
      for (int i = 0; i < kUnits; i++) k[h][i] = load_unit(keys + key * p.k.token + 32 * i + 8 * c, key < end && 32 * i + 8 * c < p.head_dim);
    }
  };
  // and of the values of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 the units g, g + 8
  constexpr int kHalves = kDim / 64;
  uint4 v[4][kHalves];
  uint32_t read = 0;                   // of these four keys
  const auto load_values = [&](int from) {
    read = 0;
#pragma unroll
    for (int h = 0; h < 4; h++) {
      const int key = from + 2 * c + (h & 1) + 8 * (h / 2);
      const bool there = key < end;
      if (there && (!mask || mask[key])) read |= 1u << h;
#pragma unroll
      for (int i = 0; i < kHalves; i++) v[h][i] = load_unit(values + key * p.v.token + 64 * i + 8 * g, there && 64 * i + 8 * g < p.head_dim);
    }
  };
  int at = first + warp * kKeys;
  load_keys(at);
  load_values(at);

  uint32_t q[2][kUnits][4];            // rows g and 8 + g, the units of the keys
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int row = row0 + 8 * h + g, token = row / p.group;
    const T* from = reinterpret_cast<const T*>(p.q.data) + batch * p.q.batch + token * p.q.token + (kv_head * p.group + row % p.group) * p.q.head;
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const uint4 x = load_unit(from + 32 * i + 8 * c, row < sp.rows && 32 * i + 8 * c < p.head_dim);
#pragma unroll
      for (int w = 0; w < 4; w++) q[h][i][w] = word_of(x, w);
    }
  }

  const float scale = p.scale * kLog2e;
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {};
  float o[kHalves][8][4] = {};
  for (; at < end; at += kWarps * kKeys) {
    float s[2][4] = {};
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < kUnits; i++) {
        const uint32_t a[4] = {q[0][i][0], q[1][i][0], q[0][i][1], q[1][i][1]}, b[4] = {q[0][i][2], q[1][i][2], q[0][i][3], q[1][i][3]};
        product16<T>(s[h], a, k[h][i].x, k[h][i].y);
        product16<T>(s[h], b, k[h][i].z, k[h][i].w);
      }
    }
    load_keys(at + kWarps * kKeys);
    // a lane has rows g (values 0, 1) and 8 + g (2, 3) of keys 2 c, 2 c + 1 and 8 more
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (!(read >> (2 * h + (e & 1)) & 1)) s[h][e] = -INFINITY;
      }
    }
    if (read != 15u) {                 // zeros where values are not read
#pragma unroll
      for (int h = 0; h < 4; h++) {
        if (!(read >> h & 1)) {
#pragma unroll
          for (int i = 0; i < kHalves; i++) v[h][i] = make_uint4(0, 0, 0, 0);
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
      for (int j = 0; j < kHalves; j++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
          for (int e = 0; e < 4; e++) o[j][i][e] *= keep[e / 2];
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
    // column n of product (j, i) is element 64 j + 8 n + i
#pragma unroll
    for (int j = 0; j < kHalves; j++) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int order = i & 1 ? 0x7632 : 0x5410;
        product16<T>(o[j][i], w, __byte_perm(word_of(v[0][j], i / 2), word_of(v[1][j], i / 2), order),
                     __byte_perm(word_of(v[2][j], i / 2), word_of(v[3][j], i / 2), order));
      }
    }
    load_values(at + kWarps * kKeys);
  }

  // the warps' sums together
#pragma unroll
  for (int r = 0; r < 2; r++) {
    total[r] += __shfl_xor_sync(~0u, total[r], 1);
    total[r] += __shfl_xor_sync(~0u, total[r], 2);
    if (c == 0) {
      warp_top[warp][8 * r + g] = top[r];
      warp_total[warp][8 * r + g] = total[r];
    }
#pragma unroll
    for (int j = 0; j < kHalves; j++) {
#pragma unroll
      for (int n = 0; n < 2; n++) {
        float* to = &warp_out[warp][8 * r + g][64 * j + 8 * (2 * c + n)];
        *reinterpret_cast<float4*>(to) = make_float4(o[j][0][2 * r + n], o[j][1][2 * r + n], o[j][2][2 * r + n], o[j][3][2 * r + n]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(o[j][4][2 * r + n], o[j][5][2 * r + n], o[j][6][2 * r + n], o[j][7][2 * r + n]);
      }
    }
  }
  __syncthreads();
  constexpr int kLanes = kDim / 8;     // threads of a row, 8 elements each
  for (int r = threadIdx.x / kLanes; r < kRows && row0 + r < sp.rows; r += 32 * kWarps / kLanes) {
    const int x = threadIdx.x % kLanes * 8, row = row0 + r, token = row / p.group, head = kv_head * p.group + row % p.group;
    float most = warp_top[0][r], sum = 0, e[8] = {};
#pragma unroll
    for (int i = 1; i < kWarps; i++) most = fmaxf(most, warp_top[i][r]);
    const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int i = 0; i < kWarps; i++) {
      const float by = exp2_of((warp_top[i][r] - base) * scale);
      sum += warp_total[i][r] * by;
#pragma unroll
      for (int j = 0; j < 8; j++) e[j] += warp_out[i][r][x + j] * by;
    }
    // only a sum of 0 is a row without keys; one that is not a number stays so, in lse too, where the joining finds it
    const float by = sum == 0 ? 0.0f : 1.0f / sum;
    const float lse = sum == 0 ? -INFINITY : most * p.scale + logf(sum);
    const int64_t stat = (static_cast<int64_t>(batch) * p.q_heads + head) * p.q_tokens + token;
    if (x < p.head_dim) {
      if (sp.splits > 1) {
        const int64_t all = static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens;
        float* to = sp.part_out + (split * all + stat) * p.head_dim + x;
        *reinterpret_cast<float4*>(to) = make_float4(e[0] * by, e[1] * by, e[2] * by, e[3] * by);
        *reinterpret_cast<float4*>(to + 4) = make_float4(e[4] * by, e[5] * by, e[6] * by, e[7] * by);
        if (x == 0) sp.part_lse[split * all + stat] = lse;
      } else {
        T* to = reinterpret_cast<T*>(p.out.data) + batch * p.out.batch + token * p.out.token + head * p.out.head + x;
        *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(e[0] * by, e[1] * by), pack2<T>(e[2] * by, e[3] * by), pack2<T>(e[4] * by, e[5] * by), pack2<T>(e[6] * by, e[7] * by));
        if (x == 0 && p.lse) p.lse[stat] = lse;
      }
    }
  }
}

// One CTA a row: its parts, weighted by exp(lse), dealt among its warps.  Sixteen where parts are many (235 parts: 18 us, four 28); four
// otherwise, whose registers fit beside the CTAs that work the parts out, so that they are there when those end (8.5 us, else 10.8).
constexpr int kManyParts = 32;

template <class T, int kJoinWarps>
__global__ void __launch_bounds__(32 * kJoinWarps) cross_join_kernel(const __grid_constant__ StepParams sp) {
  const CrossParams& p = sp.p;
  __shared__ float4 sums[kJoinWarps][32];
  __shared__ float tops[kJoinWarps], totals[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int64_t all = static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens, stat = blockIdx.x;
  const int token = stat % p.q_tokens, head = stat / p.q_tokens % p.q_heads, batch = stat / p.q_tokens / p.q_heads;
  const int parts = (length_of(p, batch) + sp.split_keys - 1) / sp.split_keys;
  wait_for_kernels_before();
  float top = -INFINITY;
  for (int i = threadIdx.x; i < parts; i += 32 * kJoinWarps) top = max_or_nan(top, sp.part_lse[i * all + stat]);
  for (int d = 16; d; d >>= 1) top = max_or_nan(top, __shfl_xor_sync(~0u, top, d));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinWarps; i++) top = max_or_nan(top, tops[i]);
  float4 o = {};
  float total = 0;
  const bool there = 4 * lane < p.head_dim;
  if (top != -INFINITY) {
#pragma unroll 4
    for (int i = warp; i < parts; i += kJoinWarps) {
      const float w = exp2_of((sp.part_lse[i * all + stat] - top) * kLog2e);
      const float4 x = there ? *reinterpret_cast<const float4*>(sp.part_out + (i * all + stat) * p.head_dim + 4 * lane) : make_float4(0, 0, 0, 0);
      total += w;
      o.x += w * x.x;
      o.y += w * x.y;
      o.z += w * x.z;
      o.w += w * x.w;
    }
  }
  sums[warp][lane] = o;
  if (lane == 0) totals[warp] = total;
  __syncthreads();
  if (warp) return;
  for (int i = 1; i < kJoinWarps; i++) {
    total += totals[i];
    o.x += sums[i][lane].x;
    o.y += sums[i][lane].y;
    o.z += sums[i][lane].z;
    o.w += sums[i][lane].w;
  }
  const float by = total == 0 ? 0.0f : 1.0f / total;
  if (there) {
    T* to = reinterpret_cast<T*>(p.out.data) + batch * p.out.batch + token * p.out.token + head * p.out.head + 4 * lane;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(o.x * by, o.y * by), pack2<T>(o.z * by, o.w * by));
  }
  if (lane == 0 && p.lse) p.lse[stat] = total == 0 ? -INFINITY : top + logf(total);
}

// Keys of a CTA: 2048 (sixteen sequences of up to 6404 keys: 57 us, with 1024 60, with 512 66), fewer (down to one round of its warps) while CTAs are fewer than two an SM, more while they are over four
// an SM and a row would have over 64 parts.
void split(const CrossParams& p, int sms, int* split_keys, int* splits) {
  const int64_t base = static_cast<int64_t>(p.batch) * p.kv_heads * ((static_cast<int64_t>(p.q_tokens) * p.group + kRows - 1) / kRows);
  int64_t keys = 2048;
  const auto parts = [&] { return (p.kv_tokens + keys - 1) / keys; };
  while (keys > kWarps * kKeys && base * parts() < 2 * sms) keys /= 2;
  while (parts() > 64 && base * parts() > 4 * sms) keys *= 2;
  *split_keys = static_cast<int>(keys);
  *splits = static_cast<int>(parts() < 1 ? 1 : parts());
}

template <class T>
cudaError_t launch(const StepParams& sp, cudaStream_t stream) {
  const CrossParams& p = sp.p;
  const dim3 grid(sp.splits, p.batch * p.kv_heads, (sp.rows + kRows - 1) / kRows);
  if (p.head_dim > 64) cross_step_kernel<T, 128><<<grid, 32 * kWarps, 0, stream>>>(sp);
  else cross_step_kernel<T, 64><<<grid, 32 * kWarps, 0, stream>>>(sp);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || sp.splits == 1) return e;
  // begins while the parts are being worked out and waits for them on the device
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(p.batch) * p.q_heads * p.q_tokens);
  const bool many = sp.splits > kManyParts;
  config.blockDim = dim3(many ? 512 : 128);
  config.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  return many ? cudaLaunchKernelEx(&config, cross_join_kernel<T, 16>, sp) : cudaLaunchKernelEx(&config, cross_join_kernel<T, 4>, sp);
}

}  // namespace

// Both ways, by what they were measured to take, in us beyond what they share: few queries 2, 1.5 for 16 rows, and keys and values once
// for every 16 rows at 4.5 TB/s; many queries 3, and 1.5 for each tile of 128 keys of each round of CTAs.  32 heads on 8, 1601 keys:
// 16 rows 10.2 and 26.1 us, 64 rows 16.3 and 26.2, 256 rows 29.1 and 26.3; 8 x 16 heads of 64, 1024 keys: 16 rows 12.5 and 15.8,
// 32 rows 20.1 and 15.8; 4 x 4 heads, 6404 keys: 64 rows 41 and 90, 256 rows 160 and 90.
bool takes_steps(const CrossParams& p, int sms) {
  const int64_t sixteens = (static_cast<int64_t>(p.q_tokens) * p.group + kRows - 1) / kRows;
  if (sixteens > 64 || static_cast<int64_t>(p.batch) * p.kv_heads > 65535) return false;
  const double bytes = 4.0 * p.batch * p.kv_heads * p.kv_tokens * p.head_dim;
  const int64_t ctas = static_cast<int64_t>(p.batch) * p.q_heads * ((p.q_tokens + 255) / 256), tiles = (p.kv_tokens + 127) / 128;
  return 2 + sixteens * (1.5 + bytes / 4.5e6) < 3 + 1.5 * ((ctas + sms - 1) / sms) * tiles;
}

size_t step_workspace(const CrossParams& p, int sms) {
  int keys, splits;
  split(p, sms, &keys, &splits);
  return splits > 1 ? sizeof(float) * splits * p.batch * p.q_heads * p.q_tokens * (p.head_dim + 1) : 0;
}

cudaError_t launch_cross_step(const CrossParams& p, void* workspace, int sms, int dtype, cudaStream_t stream) {
  StepParams sp;
  sp.p = p;
  sp.rows = p.q_tokens * p.group;
  split(p, sms, &sp.split_keys, &sp.splits);
  const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.q_tokens;
  sp.part_out = static_cast<float*>(workspace);
  sp.part_lse = sp.part_out + sp.splits * rows * p.head_dim;
  return dtype == MLXD_F16 ? launch<__half>(sp, stream) : launch<__nv_bfloat16>(sp, stream);
}

}  // namespace mlxd
