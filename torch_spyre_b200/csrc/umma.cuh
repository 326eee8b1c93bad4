// What the tcgen05 kernels share: bounded waits, moves between TMEM and registers,
// operand descriptors, the MMA instructions, packed fp32.
#pragma once

#include <type_traits>

#include "rows.cuh"

namespace b200kv {
namespace umma {

// ------------------------------------------------------------------- waits --
// Bounded: after kWaitLimitNs the error flag is set and this thread waits no
// more (its later waits return at once), so a lost transfer ends the kernel.  The
// producer then starts no more copies, and waits for those under way, with a limit
// again, before the CTA ends.
__device__ __forceinline__ void wait(uint64_t *bar, uint32_t parity, bool &dead, int32_t *flag) {
  if (mbar_try_wait(bar, parity) || dead) return;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 255u) == 0 && global_timer_ns() - t0 > kWaitLimitNs) break;
  }
  dead = true;
  if (flag) atomicOr(flag, B200KV_DEVERR_TIMEOUT);
}
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits, with a limit, until `ready` (which tests barriers side by side) holds.
template <typename Ready>
__device__ __forceinline__ void wait_until(Ready ready, bool &dead, int32_t *flag) {
  if (dead || ready()) return;
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (ready()) return;
    if ((i & 1023u) != 0) continue;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) break;
  }
  dead = true;
  if (flag) atomicOr(flag, B200KV_DEVERR_TIMEOUT);
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// -------------------------------------------------------------- TMEM moves --
#define B200KV_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), \
                        "=r"(r[i + 6]), "=r"(r[i + 7])
#define B200KV_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), \
                        "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : B200KV_R8(r, 0), B200KV_R8(r, 8), B200KV_R8(r, 16), B200KV_R8(r, 24)
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : B200KV_R8(r, 0), B200KV_R8(r, 8)
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld8(uint32_t at, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : B200KV_R8(r, 0) : "r"(at));
}
#define B200KV_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), \
                         "+r"(r[i + 6]), "+r"(r[i + 7])
// The loaded registers go through the wait, so that no use of them is moved before it.
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : B200KV_RW8(r, 0), B200KV_RW8(r, 8), B200KV_RW8(r, 16), B200KV_RW8(r, 24));
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : B200KV_RW8(r, 0), B200KV_RW8(r, 8));
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : B200KV_RW8(r, 0));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      B200KV_W8(r, 0), B200KV_W8(r, 8), B200KV_W8(r, 16), B200KV_W8(r, 24));
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;"); }
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      B200KV_W8(r, 0), B200KV_W8(r, 8));
}
__device__ __forceinline__ void tmem_st4(uint32_t at, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]));
}

// ---------------------------------------------------------------- operands --
// 128-byte swizzle, descriptor version 1.  K-major: rows of 128 bytes, groups of 8
// rows 1024 bytes apart.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // group stride, version 1, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_kmajor(uint32_t addr) { return (addr >> 4) | (1u << 16); }
// One lane of the converged warp issues (`go`); every operand is the same in
// all lanes, so that it lives in a uniform register and costs no move per MMA.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(acc), "r"(go)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(acc), "r"(go)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ void tma_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Brings `bytes` (a multiple of 16, from a 16-byte aligned address) into L2.
__device__ __forceinline__ void prefetch_l2(const void *at, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(bytes) : "memory");
}

// -------------------------------------------------------------- arithmetic --
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Softmax weights enter the tensor cores in the 16 bits of the values: 2^(y - m), off by half a
// step each (2^-8 of the weight in bf16, 2^-11 in fp16, at most), while the row's sum takes them as
// they are.  m is the running maximum less kWeightLog2, where it may lag behind by 2^8.  bf16 has
// fp32's exponents.  fp16 ends at 2^-24 below and 65504 above: with the largest weight at 1, a
// weight below 2^-25 would be lost from the products and stay in the sum, and a flat
// tail of 32768 tokens at 2^-23.5 of the loudest loses 29 % of its part.  At 2^7, and 2^15 before
// the maximum follows, what is cut off a weight is at most 2^-32 of the largest.
template <typename T>
constexpr float kWeightLog2 = std::is_same<T, __half>::value ? 7.f : 0.f;

// Two fp32 at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Non-finite elements of a vector.
// (An exponent of all ones, and no other, carries into the sign bit when its
// lowest bit is added.)
template <typename T>
__device__ __forceinline__ bool any_non_finite(uint4 v) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one)) & 0x80008000u) != 0;
}
template <typename T>
__device__ __forceinline__ uint32_t drop_non_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  if ((w & e) == e) w &= 0xffff0000u;
  if ((w & (e << 16)) == (e << 16)) w &= 0xffffu;
  return w;
}
template <typename T>
__device__ __forceinline__ bool drop_non_finite(uint4 &v) {
  const uint4 x = make_uint4(drop_non_finite<T>(v.x), drop_non_finite<T>(v.y), drop_non_finite<T>(v.z),
                             drop_non_finite<T>(v.w));
  const bool hit = x.x != v.x || x.y != v.y || x.z != v.z || x.w != v.w;
  v = x;
  return hit;
}

}  // namespace umma
}  // namespace b200kv
