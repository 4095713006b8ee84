// What the attention kernels need of sm_100a: barriers in shared memory, copies of tensor tiles, matrix products whose
// accumulators lie in tensor memory.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace mlxd {

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ---------------------------------------------------------------- barriers
__device__ __forceinline__ void barrier_init(uint32_t bar, int arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" : : "r"(bar), "r"(arrivals) : "memory");
}

__device__ __forceinline__ void barrier_init_done() {
  asm volatile("fence.mbarrier_init.release.cluster;" : : : "memory");
}

__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" : : "r"(bar) : "memory");
}

__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" : : "r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
      "selp.b32 %0, 1, 0, p;\n}"
      : "=r"(done) : "r"(bar), "r"(parity), "r"(20000) : "memory");
  return done;
}

// Every wait ends: after about two seconds (a try sleeps for 20 us at most, 4 us as measured) it sets `failed`, which ends the waits of
// the CTA's other warps too, and returns false; the caller then leaves its loop.
constexpr int kWaitTries = 500000;

__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
  if (barrier_try(bar, parity)) return true;
  for (int i = 0; i < kWaitTries; i++) {
    if (barrier_try(bar, parity)) return true;
    if (*failed) return false;
  }
  *failed = 1;
  return false;
}

// The same for a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
  return __all_sync(~0u, barrier_wait(bar, parity, failed));
}

// Where one is in a ring of kSlots slots: the slot, and the parity of its use.
template <int kSlots>
struct Ring {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void next(uint32_t by = 1) {   // by at most kSlots
    slot += by;
    if (slot >= kSlots) {
      slot -= kSlots;
      phase ^= 1;
    }
  }
};

// The same for several barriers at once: where they are ready, as they mostly are, one look costs what a look at one costs.  A barrier
// of 0 is none.
__device__ __forceinline__ bool warp_wait3(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, uint32_t bar2, uint32_t parity2, volatile int* failed) {
  const bool a = barrier_try(bar0, parity0), b = !bar1 || barrier_try(bar1, parity1), c = !bar2 || barrier_try(bar2, parity2);
  if (__all_sync(~0u, a && b && c)) return true;
  return warp_wait(bar0, parity0, failed) && (!bar1 || warp_wait(bar1, parity1, failed)) && (!bar2 || warp_wait(bar2, parity2, failed));
}

// One arrival for a warp, after what its threads did.  (An arrival of every thread is served one at a time.)
__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
  __syncwarp();
  if (lane == 0) barrier_arrive(bar);
}

// Waits for the kernels before, where this one has begun beside their end; nothing limits it, so it comes ahead of the waits that are
// limited and depend on what it waits for.
__device__ __forceinline__ void wait_for_kernels_before() {
  asm volatile("griddepcontrol.wait;" : : : "memory");
}

// Writes of this thread to shared memory are seen by copies and matrix products that are issued after this (and after a
// barrier, where another thread issues them).
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" : : : "memory");
}

// ---------------------------------------------------------------- copies of tiles: tensors are [batch][head][token][element]
__device__ __forceinline__ void tile_load(uint32_t to, const CUtensorMap* map, int element, int token, int head, int batch, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      : : "r"(to), "l"(map), "r"(element), "r"(token), "r"(head), "r"(batch), "r"(bar) : "memory");
}

__device__ __forceinline__ void tile_store(const CUtensorMap* map, int element, int token, int head, int batch, uint32_t from) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];"
               : : "l"(map), "r"(element), "r"(token), "r"(head), "r"(batch), "r"(from) : "memory");
}

__device__ __forceinline__ void tile_stores_read() {
  asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group.read 0;" : : : "memory");
}

// ---------------------------------------------------------------- tensor memory
// kColumns columns of 128 lanes of 32 bits; a whole warp allocates and frees.
template <int kColumns>
__device__ __forceinline__ void tmem_alloc(uint32_t to_smem) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" : : "r"(to_smem), "n"(kColumns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}

template <int kColumns>
__device__ __forceinline__ void tmem_free(uint32_t at) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" : : "r"(at), "n"(kColumns));
}

// kN consecutive columns of a thread's lane.  A warp reaches lanes 32 * (warp % 4) to + 31; `at` carries the first of them in its
// upper half.
template <int kN> __device__ void tmem_load(uint32_t at, uint32_t* v);
template <int kN> __device__ void tmem_store(uint32_t at, const uint32_t* v);
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(at));
}
template <>
__device__ __forceinline__ void tmem_store<16>(uint32_t at, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" : : "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(at) : "memory");
}
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]) : "r"(at));
}

// Waits for this thread's loads.  The registers they go to are named here, so that nothing that reads them is moved ahead of
// the wait: a load is under way until then, whatever the compiler thinks of its operands.
__device__ __forceinline__ void tmem_loaded(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) : : "memory");
}
__device__ __forceinline__ void tmem_loaded(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]) : : "memory");
}
__device__ __forceinline__ void tmem_loaded(uint32_t (&v)[64]) {
  tmem_loaded(reinterpret_cast<uint32_t (&)[32]>(v));
  asm volatile("" : "+r"(v[32]), "+r"(v[33]), "+r"(v[34]), "+r"(v[35]), "+r"(v[36]), "+r"(v[37]), "+r"(v[38]), "+r"(v[39]), "+r"(v[40]), "+r"(v[41]), "+r"(v[42]), "+r"(v[43]), "+r"(v[44]), "+r"(v[45]), "+r"(v[46]), "+r"(v[47]), "+r"(v[48]), "+r"(v[49]), "+r"(v[50]), "+r"(v[51]), "+r"(v[52]), "+r"(v[53]), "+r"(v[54]), "+r"(v[55]), "+r"(v[56]), "+r"(v[57]), "+r"(v[58]), "+r"(v[59]), "+r"(v[60]), "+r"(v[61]), "+r"(v[62]), "+r"(v[63]) : : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" : : : "memory"); }
__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" : : : "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" : : : "memory"); }

// ---------------------------------------------------------------- matrix products
// Tiles lie in shared memory as the copies leave them: boxes of 64 elements (128 bytes) by 128 tokens, the 16-byte units of a row
// exchanged by the row's number modulo 8 (128-byte swizzle), boxes of the elements 64 to 127 behind those of 0 to 63.
constexpr int kBoxBytes = 128 * 128;

// The constant part of a descriptor: 128-byte swizzle, version 1, 1024 bytes from eight tokens to the next eight.
// `along`: bytes to the next 64 elements where they are the operand's rows (or columns of the result) instead of what is
// summed over.
__host__ __device__ constexpr uint64_t tile_descriptor(uint32_t along) {
  return (uint64_t{2} << 61) | (uint64_t{1} << 46) | (uint64_t{1024 >> 4} << 32) | (static_cast<uint64_t>(along >> 4) << 16);
}

__device__ __forceinline__ uint64_t at_address(uint64_t descriptor, uint32_t address) {
  return descriptor | ((address & 0x3ffff) >> 4);
}

// Instruction descriptor: float32 accumulators, A and B of one 16-bit type; `b_tokens`: B is summed over its tokens (its elements
// are the columns of the result).
template <class T>
__host__ __device__ constexpr uint32_t product_descriptor(int m, int n, bool b_tokens) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | (b_tokens ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// True in one thread of a warp that runs together.  Products are issued behind this, by a warp whose threads have taken every
// branch and wait before it together.
__device__ __forceinline__ bool elected() {
  uint32_t is;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(is));
  return is;
}

// The half of a descriptor that changes: what lies `bytes` (a multiple of 16) further has `bytes >> 4` added, and nothing is carried,
// since shared memory ends below 2^18.
__device__ __forceinline__ uint32_t low_half(uint64_t descriptor) { return static_cast<uint32_t>(descriptor); }
constexpr uint32_t kHighHalf = static_cast<uint32_t>(tile_descriptor(16) >> 32);

// One product of 16 along what is summed: D (+)= A B, A and B in shared memory.
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b, uint32_t how, bool add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %5, 0;\n"
      "mov.b64 a, {%1, %4};\nmov.b64 b, {%2, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}"
      : : "r"(d), "r"(a), "r"(b), "r"(how), "r"(kHighHalf), "r"(static_cast<uint32_t>(add)) : "memory");
}

// The same with A in tensor memory, two 16-bit values a column.
__device__ __forceinline__ void product_from_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t how, bool add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %5, 0;\n"
      "mov.b64 b, {%2, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}"
      : : "r"(d), "r"(a), "r"(b), "r"(how), "r"(kHighHalf), "r"(static_cast<uint32_t>(add)) : "memory");
}

// D = A B of two tiles in shared memory, both summed over their elements, `steps` times 16 of them.
template <int kDim>
__device__ __forceinline__ void product_of_tiles(uint32_t d, uint32_t a, uint32_t b, uint32_t how, int steps) {
#pragma unroll
  for (int k = 0; k < kDim / 16; k++) {
    const uint32_t at = (k / 4 * kBoxBytes + k % 4 * 32) >> 4;
    if (k < steps) product(d, a + at, b + at, how, k > 0);
  }
}

// D (+)= A B over 64 tokens: A 128 x 64 in 32 columns of tensor memory, B half a tile summed over its tokens (the second half lies
// kHalfTokens further).
constexpr uint32_t kHalfTokens = 4 * 2048 >> 4;
__device__ __forceinline__ void product_over_tokens(uint32_t d, uint32_t a, uint32_t b, uint32_t how, bool add) {
#pragma unroll
  for (int k = 0; k < 4; k++) product_from_tmem(d, a + k * 8, b + (2048 * k >> 4), how, add || k > 0);
}

// The barrier gets an arrival when every product this thread has issued is done.
__device__ __forceinline__ void products_done(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" : : "r"(bar) : "memory");
}

// For a warp that issues products and has given up: waits, with a limit, for those under way, which read and write what the CTA is about
// to free.  `bar` is a barrier of one arrival that nothing else uses.
__device__ __forceinline__ void products_end(uint32_t bar) {
  if (elected()) products_done(bar);
  __syncwarp();
  for (int i = 0; i < kWaitTries && !barrier_try(bar, 0); i++) {}
}

// ---------------------------------------------------------------- arithmetic
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger of two; what is not a number goes on (fmaxf leaves it out).
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// a * b + c for two floats at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}

// c += a * b where `is` is not 0, by a predicate: c does not see a and b elsewhere
__device__ __forceinline__ void fma2_if(uint32_t is, float2 a, float2 b, float2& c) {
  asm("{\n.reg .pred p;\nsetp.ne.b32 p, %3, 0;\n@p fma.rn.f32x2 %0, %1, %2, %0;\n}"
      : "+l"(reinterpret_cast<uint64_t&>(c))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "r"(is));
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

// 2^x for two floats at once on the pipe of multiply-adds, which has time where the one for exponentials has not: x = n + f with n the
// nearest integer (by adding 1.5 * 2^23), 2^f = 1 + f q(f) with the cubic q of least largest relative error on [-1/2, 1/2] (2.9e-6, by
// exchange), times 2^n, whose bits are n in the exponent.  At most 2^-127 gives 0, -infinity too; what is not a number stays so, by that
// product (n added to the exponent of q would leave NaN with the bits of the largest finite number).
__device__ __forceinline__ float2 exp2_by_fma(float2 x) {
  constexpr float kRound = 12582912.0f;
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.0f));
  const float2 t = add2(x, make_float2(kRound, kRound)), n = add2(t, make_float2(-kRound, -kRound));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 q = fma2(f, make_float2(0.009582853f, 0.009582853f), make_float2(0.055906426f, 0.055906426f));
  q = fma2(f, q, make_float2(0.24024099f, 0.24024099f));
  q = fma2(f, q, make_float2(0.6931242f, 0.6931242f));
  q = fma2(f, q, make_float2(1.0f, 1.0f));
  constexpr int kOne = 127 << 23;
  return mul2(q, make_float2(__int_as_float((__float_as_int(t.x) << 23) + kOne), __int_as_float((__float_as_int(t.y) << 23) + kOne)));
}

// Two floats rounded to 16 bits each, the first in the lower half.
template <class T> __device__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// And back.
template <class T> __device__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

}  // namespace mlxd
