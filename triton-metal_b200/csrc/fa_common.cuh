// What the tcgen05 attention kernels share (fa_fwd_sm100.cu, tree_attn_sm100.cu):
// bounded waits with an abort flag, TMEM stores, the MMA forms of S = Q K^T and
// O += P V, and the softmax arithmetic (paired fp32, exponentials split
// between the MUFU unit and the FMA pipe).
#pragma once
#include "tc_common.cuh"

namespace b2 {
namespace fa {

constexpr int kF16 = 0, kBF16 = 1, kTF32 = 2;  // operand formats (tcgen05 instruction descriptor codes)

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ bool wait_abort(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code,
                                           volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitNs) break;
    }
  }
  atomicCAS(err, 0u, code);
  *abort_flag = 1;
  return false;
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem]; kind::f16 or kind::tf32 by FMT
template <int FMT>
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (FMT == kTF32) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// D[tmem] (+)= A[smem] * B[smem]^T; kind::f16 or kind::tf32 by FMT
template <int FMT>
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (FMT == kTF32) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    tc::mma_f16_ss(d_tmem, a_desc, b_desc, idesc, accumulate);
  }
}
// instruction descriptor: fp32 accumulate, A / B format FMT (0 f16, 1 bf16, 2 tf32)
__host__ __device__ constexpr uint32_t idesc_fmt(int M, int N, int fmt, bool b_mn_major) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Paired fp32 arithmetic of sm_100 (one instruction for two lanes of a
// 64-bit register pair) and the 3-input max: the softmax warps issue one
// instruction per two scores for the scale, the row sum and the max.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ float f2_lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float f2_hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// exp2 of two lanes on the FMA pipe, to take part of the softmax's
// exponentials off the MUFU unit (the method of FlashAttention-4: Cody-Waite
// split x = j + f, j = rint(x), |f| <= 1/2, then a polynomial for 2^f and j
// added into the exponent field).  The cubic is this file's own relative
// minimax fit of 2^f on [-1/2, 1/2] (max relative error 7.5e-5, below the
// 2^-9 / 2^-12 rounding of the 16-bit P it feeds).  x <= 8 here; x is clamped
// at -125 so that 2^j stays a normal number.
__device__ __forceinline__ uint64_t exp2_poly_f2(uint64_t x2) {
  const uint64_t x = f2_pack(fmaxf(f2_lo(x2), -125.f), fmaxf(f2_hi(x2), -125.f));
  const float kRound = 12582912.f;  // 1.5 * 2^23: x + kRound rounds x to an integer in the low mantissa bits
  const uint64_t t = add_f2(x, f2_pack(kRound, kRound));
  const uint64_t j = add_f2(t, f2_pack(-kRound, -kRound));
  const uint64_t fr = fma_f2(j, f2_pack(-1.f, -1.f), x);
  uint64_t q = fma_f2(f2_pack(0.05517132f, 0.05517132f), fr, f2_pack(0.24261054f, 0.24261054f));
  q = fma_f2(q, fr, f2_pack(0.69326097f, 0.69326097f));
  q = fma_f2(q, fr, f2_pack(0.99992812f, 0.99992812f));
  // bits(t) = 0x4B400000 + j, so bits(t) << 23 = j << 23 (mod 2^32)
  const uint32_t lo = (uint32_t)t * (1u << 23) + (uint32_t)q;
  const uint32_t hi = (uint32_t)(t >> 32) * (1u << 23) + (uint32_t)(q >> 32);
  return (uint64_t)lo | ((uint64_t)hi << 32);
}

}  // namespace fa
}  // namespace b2
