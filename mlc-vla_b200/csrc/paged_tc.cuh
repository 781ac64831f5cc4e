// Tensor-core pieces shared by the attention kernels over prompts and over the cache: matrix
// descriptors for every swizzle, the 8-bit MMA, TMEM access of other widths, 3-D TMA loads.
#pragma once

#include "gemm_tc.cuh"

namespace pi0 {
namespace paged {

using tc::globaltimer;
using tc::mbar_arrive;
using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::tc_fence_after;
using tc::tc_fence_before;
using tc::tma_prefetch_desc;
using tc::tmem_ld32;
using tc::umma_commit;

// Byte offset inside a tile of `row_bytes`-wide rows (32, 64 or 128, the swizzle span) after the
// swizzle that TMA and the matrix descriptors use: the 16-byte chunk index is XORed with the
// address bits from 128 bytes up.
template <int ROW>
__device__ __forceinline__ uint32_t swz(uint32_t off) {
  constexpr uint32_t mask = ROW / 16 - 1;
  return off ^ (((off >> 7) & mask) << 4);
}

// Shared-memory matrix descriptor of an operand in rows of `ROW` bytes, swizzled over that span.
// K-major: sbo = bytes between groups of 8 rows. MN-major: sbo = bytes between groups of 8 k,
// lbo = bytes between ROW-wide blocks along m or n.
template <int ROW>
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t sbo, uint32_t lbo) {
  constexpr uint64_t layout = ROW == 128 ? 2 : ROW == 64 ? 4 : 6;
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;
  d |= layout << 61;
  return d;
}

// kind::f8f6f4: e4m3 operands (format 0), fp32 accumulator
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// kind::f16 with A in tensor memory (each 32-bit column holds two consecutive k of a lane's row)
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t b,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate));
}

// tmem_ld32 without the wait: the values may be used after tmem_wait_ld
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 lanes × 32 columns, the store that mirrors tmem_ld32 (no wait)
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld32(taddr, r);
}
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  tmem_wait_ld();
}
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[32]) {
  tmem_st32(taddr, r);
}
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[16]) {
  tmem_st16(taddr, r);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x,
                                            int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Bounded waits of one CTA (about a second of globaltimer each). One that gives up records its code
// for the call and sets the CTA's `stop`, at which its other waits give up as well. They do not look
// at *err: it may hold what an earlier call or another request has recorded.
struct Waits {
  int* err;
  volatile int* stop;  // shared memory, zero at the start
};
__device__ __forceinline__ bool wait_polling(uint64_t* bar, uint32_t parity, const Waits& w, int code,
                                             bool bail) {
  const unsigned long long t0 = globaltimer();
  for (uint32_t it = 1;; ++it) {
    if (tc::mbar_try(bar, parity)) return true;
    if ((it & 127) == 0) {
      if (bail && *w.stop) return false;
      if (globaltimer() - t0 > tc::kTimeoutNs) {
        atomicCAS(w.err, 0, code);
        *w.stop = 1;
        return false;
      }
    }
  }
}
static __device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, Waits w, int code,
                                              bool bail) {
  return wait_polling(bar, parity, w, code, bail);
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, const Waits& w, int code,
                                          bool bail = true) {
  if (tc::mbar_try(bar, parity)) return true;
  return wait_slow(bar, parity, w, code, bail);
}
// the same without a call, for kernels that shift registers between warps (setmaxnreg allows none)
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, const Waits& w, int code,
                                         bool bail = true) {
  if (tc::mbar_try(bar, parity)) return true;
  return wait_polling(bar, parity, w, code, bail);
}

// One thread of a converged warp. Tensor-core instructions are issued by a whole warp's control flow
// under this predicate: their operands then stay in uniform registers. From a branch on the lane
// number each of them took over 100 clocks to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(r));
  return r != 0;
}

// `total` pieces of work, numbered in one row, in contiguous shares of `each` or, the first `extra`
// ones, one more; no share is empty, so fewer pieces than CTAs leave the last CTAs without one.
template <typename I>
struct Shares {
  I each, extra;
  __device__ __forceinline__ Shares(I total, int ctas) {
    const I some = max((I)1, min(total, (I)ctas));
    each = total / some;
    extra = total - each * some;
  }
  __device__ __forceinline__ I begin(int cta, I total) const {
    return min(total, cta * each + min((I)cta, extra));
  }
  __device__ __forceinline__ int owner(I at) const {
    const I wide = extra * (each + 1);
    return (int)(at < wide ? at / (each + 1) : extra + (at - wide) / each);
  }
};

// ---- two fp32 at a time: the packed forms issue once for both ----
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// largest of a warp's values (NaN counts as smaller), one instruction
__device__ __forceinline__ float warp_max_f32(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// whether any of the block's N threads says so; warps may come to it from different places
template <int N>
__device__ __forceinline__ bool block_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 0, %2, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)v), "n"(N)
      : "memory");
  return r != 0;
}

template <int ID, int N>
__device__ __forceinline__ void named_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}

}  // namespace paged
}  // namespace pi0
