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

// ---------------------------------------------------------------------------
// Scores with a mask of one bit per key, a cap and a distance bias, for one
// 128-key tile; this thread's row is its TMEM lane.  In log2 units:
//   x = scale s            or  x = cap tanh(scale s / cap)
//   x -= slope |row - key|
// ---------------------------------------------------------------------------
struct Score {
  float scale_log2;        // scale * log2 e (> 0)
  float cap_in, cap_log2;  // 2 log2 e scale / cap; cap * log2 e
  float slope, dist;       // slope * log2 e; row - first key of the tile
};

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap tanh(scale s / cap) + add: tanh y = 1 - 2 / (1 + e^2y), good to ~2e-7
// (the one-instruction tanh is good to 2^-11, which a cap of 50 turns into 0.02
// in the exponent)
__device__ __forceinline__ float capped(float s, const Score& c, float add) {
  return fmaf(-2.f * c.cap_log2, rcp_approx(1.f + ex2(s * c.cap_in)), c.cap_log2 + add);
}

// Score of two neighbouring keys (e and e + 1 in the tile), plus `add`.  Where
// MASK is false all keys of the tile lie on one side of the row, so the bias is
// linear in the key: slope carries its sign there (slope > 0: keys before the
// row).
template <bool MASK, bool CAP, bool BIAS>
__device__ __forceinline__ uint64_t score_pair(uint32_t s0, uint32_t s1, int e, const Score& c, float add) {
  uint64_t a = f2_pack(add, add);
  if constexpr (BIAS) {
    if constexpr (MASK) {
      a = f2_pack(fmaf(-c.slope, fabsf(c.dist - (float)e), add), fmaf(-c.slope, fabsf(c.dist - (float)(e + 1)), add));
    } else {
      const float b = fmaf(-c.slope, c.dist, add);
      a = fma_f2(f2_pack(c.slope, c.slope), f2_pack((float)e, (float)(e + 1)), f2_pack(b, b));
    }
  }
  if constexpr (CAP)
    return f2_pack(capped(__uint_as_float(s0), c, f2_lo(a)), capped(__uint_as_float(s1), c, f2_hi(a)));
  return fma_f2((uint64_t)s0 | ((uint64_t)s1 << 32), f2_pack(c.scale_log2, c.scale_log2), a);
}

// Largest score of the row's visible keys (bits of vis), -inf without one.
// Scale and cap keep the order, so without a bias the raw maximum is taken and
// scored once.  With cap and bias both, the scores are left in the S columns
// for score_exp, so that the cap is computed once.
template <bool MASK, bool CAP, bool BIAS>
__device__ __forceinline__ float score_max(uint32_t tS, const uint32_t (&vis)[4], const Score& sc) {
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    uint32_t sv[64];
    tc::tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
    tc::tmem_ld_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
    tc::tmem_ld_wait();
    const uint32_t w0 = c ? vis[2] : vis[0], w1 = c ? vis[3] : vis[1];
    Score cc = sc;
    cc.dist -= 32.f * c;
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
      float v0 = __uint_as_float(sv[e]), v1 = __uint_as_float(sv[e + 1]);
      if constexpr (BIAS) {
        const uint64_t x = score_pair<MASK, CAP, BIAS>(sv[e], sv[e + 1], e, cc, 0.f);
        v0 = f2_lo(x);
        v1 = f2_hi(x);
        if constexpr (CAP) {
          sv[e] = (uint32_t)x;
          sv[e + 1] = (uint32_t)(x >> 32);
        }
      }
      if constexpr (MASK) {
        const uint32_t w = e < 32 ? w0 : w1;
        if (!(w >> (e & 31) & 1)) v0 = -INFINITY;
        if (!(w >> ((e + 1) & 31) & 1)) v1 = -INFINITY;
      }
      mx = max3(mx, v0, v1);
    }
    if constexpr (CAP && BIAS) {
      tmem_st_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
      tmem_st_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
    }
  }
  if constexpr (CAP && BIAS) tmem_st_wait();
  if constexpr (!BIAS) {
    if constexpr (CAP) mx = mx == -INFINITY ? mx : capped(mx, sc, 0.f);
    else mx *= sc.scale_log2;
  }
  return mx;
}

// p = exp2(score - m) as 16-bit pairs over the S columns; returns their sum.
// P rounded to 16 bits (half a step of its own size) is what the MMA takes; the
// sum is taken before that, in 32 bits.
template <bool MASK, int FMT, bool CAP, bool BIAS>
__device__ __forceinline__ float score_exp(uint32_t tS, const uint32_t (&vis)[4], float mref, const Score& sc) {
  uint64_t rs = 0;
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    uint32_t sv[64];
    tc::tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
    tc::tmem_ld_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
    tc::tmem_ld_wait();
    const uint32_t w0 = c ? vis[2] : vis[0], w1 = c ? vis[3] : vis[1];
    Score cc = sc;
    cc.dist -= 32.f * c;
    uint32_t pk[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      float p0, p1;
      uint64_t x;
      if constexpr (CAP && BIAS) x = add_f2((uint64_t)sv[2 * e] | ((uint64_t)sv[2 * e + 1] << 32), f2_pack(-mref, -mref));
      else x = score_pair<MASK, CAP, BIAS>(sv[2 * e], sv[2 * e + 1], 2 * e, cc, -mref);
      if (e % 3 == 2) {  // a third of the exponentials on the FMA pipe, as in the prefill kernel
        const uint64_t y = exp2_poly_f2(x);
        p0 = f2_lo(y);
        p1 = f2_hi(y);
      } else {
        p0 = ex2(f2_lo(x));
        p1 = ex2(f2_hi(x));
      }
      if constexpr (MASK) {
        const uint32_t w = e < 16 ? w0 : w1;
        if (!(w >> ((2 * e) & 31) & 1)) p0 = 0.f;
        if (!(w >> ((2 * e + 1) & 31) & 1)) p1 = 0.f;
      }
      rs = add_f2(rs, f2_pack(p0, p1));
      if constexpr (FMT == kF16) {
        __half2 hv = __floats2half2_rn(p0, p1);
        pk[e] = *reinterpret_cast<uint32_t*>(&hv);
      } else {
        __nv_bfloat162 hv = __floats2bfloat162_rn(p0, p1);
        pk[e] = *reinterpret_cast<uint32_t*>(&hv);
      }
    }
    tmem_st_32x32b_x32(tS + 16 * c, pk);
  }
  return f2_lo(rs) + f2_hi(rs);
}

template <int FMT>
__device__ __forceinline__ bool not_finite16(uint32_t h) {  // of the low half
  constexpr uint32_t e = FMT == kF16 ? 0x7C00u : 0x7F80u;
  return (h & e) == e;
}
// Zeroes the 16-bit values of a chunk that are infinite or NaN; true if there were any.
template <int FMT>
__device__ __forceinline__ bool zero_not_finite(uint4& x) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&x);
  bool hit = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (not_finite16<FMT>(w[e])) w[e] &= 0xffff0000u, hit = true;
    if (not_finite16<FMT>(w[e] >> 16)) w[e] &= 0x0000ffffu, hit = true;
  }
  return hit;
}
template <int FMT>
__device__ __forceinline__ float widen16(uint16_t h) {
  if constexpr (FMT == kF16) return __half2float(__ushort_as_half(h));
  else return __uint_as_float((uint32_t)h << 16);
}
template <int FMT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (FMT == kF16) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

}  // namespace fa
}  // namespace b2
