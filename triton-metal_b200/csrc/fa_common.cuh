// What the tcgen05 attention kernels share (fa_fwd_sm100.cu, tree_attn_sm100.cu):
// bounded waits with an abort flag, TMEM stores, the MMA forms of S = Q K^T and
// O += P V, and the softmax arithmetic (paired fp32, exponentials split
// between the MUFU unit and the FMA pipe).
#pragma once
#include "tc_common.cuh"
#include <string.h>

namespace b2 {
namespace fa {

constexpr int kF16 = 0, kBF16 = 1, kTF32 = 2;  // operand formats (tcgen05 instruction descriptor codes)
constexpr int BQ = 128, BKV = 128;
constexpr int kKStages = 3, kVStages = 2;

// Tile geometry of the tcgen05 path for head dim HD and operand format FMT
// (kTF32: fp32 q / k / v read as tf32, fp32 output).  A tile is BQ rows of HD
// elements in 128-byte swizzle atoms; one MMA k-step is 32 bytes of K.
template <int HD_, int FMT_>
struct FaCfg {
  static constexpr int HD = HD_, FMT = FMT_;
  static constexpr int ES = FMT == kTF32 ? 4 : 2;   // element bytes
  static constexpr int KSTEP = 32 / ES;             // K elements per MMA
  static constexpr int AE = 128 / ES;               // elements per swizzle row
  static constexpr int NATOM = HD / AE;
  static constexpr int kAtom = BQ * 128;            // bytes of one atom column
  static constexpr int kTile = NATOM * kAtom;
  static constexpr size_t kSmem = (size_t)kTile * (2 + kKStages + kVStages) + 1024 + 256;
  static_assert(HD % AE == 0, "head dim must fill whole swizzle rows");
};

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
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if one of them is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
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
  float small;             // scores up to this size take capped_small (negative: none)
  uint64_t t[5], scale2;   // its coefficients and scale_log2, each twice
  float slope, dist;       // slope * log2 e (score_pair: with a side's sign); row - first key of the tile
  float slope0;            // slope * log2 e as given, of either sign
};

// What a kernel's parameters hold of it.  The operands of the paired instructions
// lie there as pairs, so that they are read from constant memory; pairs made in
// registers cost a move or two at every use.
struct Cap {
  float scale_log2, in, log2, small;
  uint64_t t[5], scale2;
};
__device__ __forceinline__ Score make_score(const Cap& c) {
  return {c.scale_log2, c.in, c.log2, c.small, {c.t[0], c.t[1], c.t[2], c.t[3], c.t[4]}, c.scale2, 0.f, 0.f, 0.f};
}
// key numbers of a piece, for the distance bias
__device__ __constant__ const float2 kKeys[32] = {
    {0, 1},   {2, 3},   {4, 5},   {6, 7},   {8, 9},   {10, 11}, {12, 13}, {14, 15}, {16, 17}, {18, 19}, {20, 21},
    {22, 23}, {24, 25}, {26, 27}, {28, 29}, {30, 31}, {32, 33}, {34, 35}, {36, 37}, {38, 39}, {40, 41}, {42, 43},
    {44, 45}, {46, 47}, {48, 49}, {50, 51}, {52, 53}, {54, 55}, {56, 57}, {58, 59}, {60, 61}, {62, 63}};
// tanh z = z p(z^2) on [-3/4, 3/4]: this file's own minimax fit (largest error
// 2.4e-7 in fp32).  The coefficients take scale, cap and log2 e with them, so
// that a score s gives s q(s^2).  The powers of scale / cap have to stay in
// fp32's range: above 1e3 the form is not used, and below 2e-4 (caps so high that
// hardly a score feels them) only up to z = 0.05, where the first three terms
// are enough: the other form's error, a part of the cap, would drown the scores.
inline Cap make_cap(float scale, float softcap) {
  Cap c = {};
  auto twice = [](float x) {
    uint32_t u;
    memcpy(&u, &x, 4);
    return (uint64_t)u << 32 | u;
  };
  c.scale_log2 = scale * 1.4426950408889634f;
  c.scale2 = twice(c.scale_log2);
  c.small = -1.f;
  if (softcap > 0.f) {
    const double log2e = 1.4426950408889634, z = (double)scale / softcap;
    const double p[5] = {0.9999971985816956, -0.33323076367378235, 0.13226091861724854, -0.04928044602274895,
                         0.012318830005824566};
    c.in = (float)fmin(2 * log2e * z, 1e37);  // 0 times it is 0
    c.log2 = (float)(log2e * softcap);
    if (z > 1e3) return c;
    c.small = (float)(z > 2e-4 ? 0.75 / z : fmin(0.05 / z, 1e18));
    double f = log2e * softcap * z;
    for (int i = 0; i < (z > 2e-4 ? 5 : 3); ++i, f *= z * z) c.t[i] = twice((float)(p[i] * f));
  }
  return c;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// cap tanh(scale s / cap) + add: tanh y = 1 - 2 / (1 + e^2y), good to ~2e-7
// (the one-instruction tanh is good to 2^-11, which a cap of 50 turns into 0.02
// in the exponent)
__device__ __forceinline__ float capped(float s, const Score& c, float add) {
  return fmaf(-2.f * c.cap_log2, rcp_approx(1.f + ex2(s * c.cap_in)), c.cap_log2 + add);
}
// The same for two scores of at most c.small, on the FMA pipe: the two MUFU
// operations a score of the form above would set the pace of the softmax.
__device__ __forceinline__ uint64_t capped_small(uint64_t s, const Score& c, uint64_t add) {
  const uint64_t w = mul_f2(s, s);
  uint64_t q = fma_f2(c.t[4], w, c.t[3]);
  q = fma_f2(q, w, c.t[2]);
  q = fma_f2(q, w, c.t[1]);
  q = fma_f2(q, w, c.t[0]);
  return fma_f2(s, q, add);
}
__device__ __forceinline__ float capped_any(float s, const Score& c, float add) {
  if (fabsf(s) <= c.small) return f2_lo(capped_small(f2_pack(s, s), c, f2_pack(add, add)));
  return capped(s, c, add);
}
// Whether all of the warp's N x 32 scores may take capped_small (w: 0 where the
// row sees none of them).
template <int N>
__device__ __forceinline__ bool all_small(const uint32_t (&sv)[N], uint32_t w, const Score& c) {
  float am = 0.f;
#pragma unroll
  for (int e = 0; e < N; e += 2) am = max3(am, fabsf(__uint_as_float(sv[e])), fabsf(__uint_as_float(sv[e + 1])));
  return !__any_sync(0xffffffffu, w && !(am <= c.small));
}

// Score of two neighbouring keys (e and e + 1 from where c.dist counts), plus
// `add`.  ABS: keys on both sides of the row.  Otherwise all keys of the tile
// lie on one side, the bias is linear in the key and c.slope is the slope where
// they are before the row, minus the slope where they are behind it.
template <bool ABS, bool CAP, bool BIAS, bool SMALL>
__device__ __forceinline__ uint64_t score_pair(uint32_t s0, uint32_t s1, int e, const Score& c, float add) {
  uint64_t a = f2_pack(add, add);
  if constexpr (BIAS) {
    if constexpr (ABS) {
      const float sl = -c.slope0;
      a = f2_pack(fmaf(sl, fabsf(c.dist - (float)e), add), fmaf(sl, fabsf(c.dist - (float)(e + 1)), add));
    } else {
      const float b = fmaf(-c.slope, c.dist, add);
      a = fma_f2(f2_pack(c.slope, c.slope), f2_pack(kKeys[e / 2].x, kKeys[e / 2].y), f2_pack(b, b));
    }
  }
  const uint64_t s = (uint64_t)s0 | ((uint64_t)s1 << 32);
  if constexpr (CAP && SMALL) return capped_small(s, c, a);
  if constexpr (CAP)
    return f2_pack(capped(__uint_as_float(s0), c, f2_lo(a)), capped(__uint_as_float(s1), c, f2_hi(a)));
  return fma_f2(s, c.scale2, a);
}

// Scores of the N columns in sv, left in sv (with a bias, which the maximum
// needs too).
template <bool ABS, bool CAP, bool SMALL, int N>
__device__ __forceinline__ void score_chunk(uint32_t (&sv)[N], const Score& c) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const uint64_t x = score_pair<ABS, CAP, true, SMALL>(sv[e], sv[e + 1], e, c, 0.f);
    sv[e] = (uint32_t)x;
    sv[e + 1] = (uint32_t)(x >> 32);
  }
}

// Largest of N columns, NaN if one of them is; BITS: of those with a bit in w (N = 32).
template <bool BITS, int N>
__device__ __forceinline__ float max_chunk(const uint32_t (&sv)[N], uint32_t w) {
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    float v0 = __uint_as_float(sv[e]), v1 = __uint_as_float(sv[e + 1]);
    if constexpr (BITS) {
      if (!(w >> e & 1)) v0 = -INFINITY;
      if (!(w >> (e + 1) & 1)) v1 = -INFINITY;
    }
    mx = max3_nan(mx, v0, v1);
  }
  return mx;
}

// A tile that each of the warp's rows sees whole or not at all is gone through
// in halves of 64 keys (WIDE; two TMEM loads a wait), another one in four pieces of
// 32.  Of those, one that each row sees whole or not at all (and, with a bias,
// whose keys lie on one side of the rows) takes the short way too, one that
// nobody sees is passed over, and the rest are masked by bits.  So a document's
// border costs little in the many tiles that lie to one side of it.
enum Piece { kNone, kRows, kBits };
__device__ __forceinline__ Piece piece_of(uint32_t w, bool rows_ok) {
  if (!__any_sync(0xffffffffu, w != 0)) return kNone;
  return rows_ok && __all_sync(0xffffffffu, w == 0 || w == 0xffffffffu) ? kRows : kBits;
}
__device__ __forceinline__ uint32_t word_of(const uint32_t (&vis)[4], int c) {
  return c == 0 ? vis[0] : c == 1 ? vis[1] : c == 2 ? vis[2] : vis[3];
}
// each of the warp's rows sees all 128 keys or none (vis[0] says which)
__device__ __forceinline__ bool whole_tile(const uint32_t (&vis)[4]) {
  return __all_sync(0xffffffffu, (vis[0] & vis[1] & vis[2] & vis[3]) == 0xffffffffu ||
                                     (vis[0] | vis[1] | vis[2] | vis[3]) == 0);
}

// p = exp2(score - m) of N columns as 16-bit pairs; returns their sum.
template <bool BITS, int FMT, bool CAP, bool BIAS, bool SMALL, int N>
__device__ __forceinline__ float exp_chunk(const uint32_t (&sv)[N], uint32_t (&pk)[N / 2], uint32_t w, const Score& c,
                                           float mref) {
  uint64_t rs = 0;
#pragma unroll
  for (int e = 0; e < N / 2; ++e) {
    float p0, p1;
    uint64_t x;
    if constexpr (BIAS) x = add_f2((uint64_t)sv[2 * e] | ((uint64_t)sv[2 * e + 1] << 32), f2_pack(-mref, -mref));
    else x = score_pair<BITS, CAP, BIAS, SMALL>(sv[2 * e], sv[2 * e + 1], 2 * e, c, -mref);
    // part of the exponentials on the FMA pipe: a third, as in the prefill
    // kernel, but fewer beside the cap, which has filled it already
    if (CAP ? e % 8 == 7 : e % 3 == 2) {
      const uint64_t y = exp2_poly_f2(x);
      p0 = f2_lo(y);
      p1 = f2_hi(y);
    } else {
      p0 = ex2(f2_lo(x));
      p1 = ex2(f2_hi(x));
    }
    if constexpr (BITS) {
      if (!(w >> (2 * e) & 1)) p0 = 0.f;
      if (!(w >> (2 * e + 1) & 1)) p1 = 0.f;
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
  return f2_lo(rs) + f2_hi(rs);
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
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

// The running maximum has grown: O (HD columns, if there is one yet) and the P
// of the keys [from, to), which this tile has stored already, are brought to the
// new one.  Both may still be on their way to TMEM, O from an earlier rescaling of
// the same tile, and nothing orders a load behind a store but the wait.
template <int HD, int FMT>
__device__ __forceinline__ void rescale(uint32_t tO, uint32_t tP, bool has_o, int from, int to, float alpha) {
  tmem_st_wait();
  if (has_o) {
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t o[32];
      tc::tmem_ld_32x32b_x32(tO + 32 * c, o);
      tc::tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
      tmem_st_32x32b_x32(tO + 32 * c, o);
    }
  }
  if (from < to) {
#pragma unroll 1
    for (int c = from / 32; c < to / 32; ++c) {
      uint32_t x[16];
      tmem_ld_32x32b_x16(tP + 16 * c, x);
      tc::tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e)
        x[e] = narrow2<FMT>(widen16<FMT>((uint16_t)x[e]) * alpha, widen16<FMT>((uint16_t)(x[e] >> 16)) * alpha);
      tmem_st_32x32b_x16(tP + 16 * c, x);
    }
  }
}

// First column of P (64 columns) among the 128 of S: P of a piece must only
// cover columns of S that are read already, from the left when the keys are
// taken from first to last, from the right when they are taken from last to
// first.
__host__ __device__ constexpr int p_column(bool last_first) { return last_first ? 64 : 0; }

constexpr float kRescale = 8.f;  // log2 units: P holds up to 2^8

// 2^d for a whole d <= 0 (-inf: 0)
__device__ __forceinline__ float pow2_down(float d) {
  return d < -126.f ? 0.f : __int_as_float((int)(d + 127.f) << 23);
}

// One chunk of a tile (N = 64 or 32 keys from key `at` on): its maximum, the
// rescaling if that has grown by more than kRescale, and its P over the S
// columns.  w: BITS, a bit per key; else all ones or zero, the row sees the
// chunk or not.
template <bool BITS, int HD, int FMT, bool CAP, bool BIAS, int N>
__device__ __forceinline__ void softmax_chunk(uint32_t (&sv)[N], uint32_t tS, uint32_t tO, int at, uint32_t w,
                                              const Score& sc, bool has_o, float& m, float& l) {
  Score cc = sc;
  cc.dist -= (float)at;
  bool small = false;
  if constexpr (CAP) small = all_small(sv, w, sc);
  if constexpr (BIAS) {
    if (CAP && small) score_chunk<BITS, CAP, CAP>(sv, cc);
    else score_chunk<BITS, CAP, false>(sv, cc);
  }
  float mx = max_chunk<BITS>(sv, w);
  if constexpr (!BIAS) {  // scale and cap keep the order
    if constexpr (CAP) mx = mx == -INFINITY ? mx : capped_any(mx, sc, 0.f);
    else mx *= sc.scale_log2;
  }
  if (!BITS && !w) mx = -INFINITY;
  // a score that is NaN, or infinite (inf - inf), makes NaN of the row; where its
  // exponential is the polynomial's, that would lose it
  if (!(mx < INFINITY)) l = NAN;
  const bool need = mx > m + kRescale;
  if (__any_sync(0xffffffffu, need)) {
    // the first maximum as it is (a row's only key has weight 1), then whole steps
    // up from it: what is stored as P already is rescaled exactly, and no weight
    // is rounded twice
    const float up = ceilf(mx - m);
    const float alpha = need ? pow2_down(-up) : 1.f;
    if (need) {
      l *= alpha;
      m = m == -INFINITY ? mx : m + up;
    }
    rescale<HD, FMT>(tO, tS + p_column(BIAS), has_o, BIAS ? at + N : 0, BIAS ? 128 : at, alpha);
  }
  const float mref = m == -INFINITY ? 0.f : m;
  uint32_t pk[N / 2];
  float rs;
  if (CAP && !BIAS && small) rs = exp_chunk<BITS, FMT, CAP, BIAS, CAP && !BIAS>(sv, pk, w, cc, mref);
  else rs = exp_chunk<BITS, FMT, CAP, BIAS, false>(sv, pk, w, cc, mref);
  if constexpr (!BITS) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) pk[e] &= w;
    if (!w) rs = 0.f;
  }
  l += rs;
  if constexpr (N == 64) tmem_st_32x32b_x32(tS + p_column(BIAS) + at / 2, pk);
  else tmem_st_32x32b_x16(tS + p_column(BIAS) + at / 2, pk);
}

// The softmax of one tile in a single pass over S: P = exp2(score - m) as 16-bit
// pairs over the S columns, m and l brought up to date, O (has_o: there is one)
// rescaled where the maximum has grown by more than kRescale.  P rounded to 16
// bits (half a step of its own size) is what the MMA takes; the sum l is taken
// before that, in 32 bits.
// With a bias the keys are taken from the last to the first (and the tiles, by
// the callers): the nearer a key, the larger its score, so that the maximum is
// found at once instead of growing with every piece.
// vis: a bit per key.  WIDE: with the way for whole tiles, taken where `whole`
// says so (whole_tile, and with a bias all keys on one side); one_side: see
// score_pair.
template <bool WIDE, int HD, int FMT, bool CAP, bool BIAS>
__device__ __forceinline__ void softmax_tile(uint32_t tS, uint32_t tO, const uint32_t (&vis)[4], bool whole,
                                             bool one_side, const Score& sc, bool has_o, float& m, float& l) {
  if (WIDE && whole) {
#pragma unroll 1
    for (int i = 0; i < 4; i += 2) {
      const int c = BIAS ? 2 - i : i;
      uint32_t sv[64];
      tc::tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
      tc::tmem_ld_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
      tc::tmem_ld_wait();
      softmax_chunk<false, HD, FMT, CAP, BIAS>(sv, tS, tO, 32 * c, vis[0], sc, has_o, m, l);
    }
    return;
  }
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int c = BIAS ? 3 - i : i;
    const uint32_t w = word_of(vis, c);
    const Piece kind = piece_of(w, !BIAS || one_side);
    if (kind == kNone) {
      uint32_t zero[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) zero[e] = 0;
      tmem_st_32x32b_x16(tS + p_column(BIAS) + 16 * c, zero);
      continue;
    }
    uint32_t sv[32];
    tc::tmem_ld_32x32b_x32(tS + 32 * c, sv);
    tc::tmem_ld_wait();
    if (kind == kRows) softmax_chunk<false, HD, FMT, CAP, BIAS>(sv, tS, tO, 32 * c, w, sc, has_o, m, l);
    else softmax_chunk<true, HD, FMT, CAP, BIAS>(sv, tS, tO, 32 * c, w, sc, has_o, m, l);
  }
}

// The same for a warp whose 32 rows are at most 8 (rows 0 to 7, its TMEM lanes)
// and that takes 32 keys of the tile only, those of piece `piece` (its P is 0 for
// the others): four lanes a row with 8 keys each, instead of 32 keys in each of a
// few lanes.  Scores and weights change lanes through 1 KB of shared memory.  w:
// keys that row `lane` sees; m and l: of row lane % 8, l of this lane's keys.
template <int HD, int FMT, bool CAP, bool BIAS>
__device__ __forceinline__ void softmax_few(uint8_t* room, uint32_t tS, uint32_t tO, int piece, uint32_t w,
                                            const Score& sc, bool has_o, float& m, float& l) {
  const int lane = threadIdx.x & 31, row = lane & 7, part = lane >> 3;
  uint32_t sv[8];
  {
    uint32_t all[32];
    tc::tmem_ld_32x32b_x32(tS + 32 * piece, all);
    tc::tmem_ld_wait();
    __syncwarp();  // the tile before is read
    if (lane < 8) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<uint4*>(room + row * 128 + ((c ^ row) << 4)) =
            make_uint4(all[4 * c], all[4 * c + 1], all[4 * c + 2], all[4 * c + 3]);
    }
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint4 x = *reinterpret_cast<const uint4*>(room + row * 128 + (((2 * part + c) ^ row) << 4));
    sv[4 * c] = x.x;
    sv[4 * c + 1] = x.y;
    sv[4 * c + 2] = x.z;
    sv[4 * c + 3] = x.w;
  }
  const uint32_t bits = __shfl_sync(0xffffffffu, w, row) >> (8 * part) & 0xffu;
  Score cc = sc;
  cc.dist -= (float)(32 * piece + 8 * part);
  bool small = false;
  if constexpr (CAP) small = all_small(sv, bits, sc);
  if constexpr (BIAS) {
    cc.slope = __shfl_sync(0xffffffffu, sc.slope, row);
    if (CAP && small) score_chunk<false, CAP, CAP>(sv, cc);
    else score_chunk<false, CAP, false>(sv, cc);
  }
  float mx = max_chunk<true>(sv, bits);
  if constexpr (!BIAS) {
    if constexpr (CAP) mx = mx == -INFINITY ? mx : capped_any(mx, sc, 0.f);
    else mx *= sc.scale_log2;
  }
  if (!(mx < INFINITY)) l = NAN;  // as in softmax_chunk; this lane's part of the row's sum
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
  const bool need = mx > m + kRescale;
  if (__any_sync(0xffffffffu, need)) {  // as in softmax_chunk
    const float up = ceilf(mx - m);
    const float alpha = need ? pow2_down(-up) : 1.f;
    if (need) {
      l *= alpha;
      m = m == -INFINITY ? mx : m + up;
    }
    rescale<HD, FMT>(tO, 0, has_o, 0, 0, alpha);
  }
  const float mref = m == -INFINITY ? 0.f : m;
  uint32_t pk[4];
  if (CAP && !BIAS && small) l += exp_chunk<true, FMT, CAP, BIAS, CAP && !BIAS>(sv, pk, bits, cc, mref);
  else l += exp_chunk<true, FMT, CAP, BIAS, false>(sv, pk, bits, cc, mref);
  __syncwarp();  // the scores are read
  *reinterpret_cast<uint4*>(room + row * 64 + ((part ^ (row >> 1 & 3)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
  __syncwarp();
  uint32_t p[16];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 x = *reinterpret_cast<const uint4*>(room + row * 64 + ((c ^ (row >> 1 & 3)) << 4));
    p[4 * c] = lane < 8 ? x.x : 0;
    p[4 * c + 1] = lane < 8 ? x.y : 0;
    p[4 * c + 2] = lane < 8 ? x.z : 0;
    p[4 * c + 3] = lane < 8 ? x.w : 0;
  }
  uint32_t zero[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) zero[e] = 0;
#pragma unroll 1
  for (int c = 0; c < 4; ++c)
    if (c != piece) tmem_st_32x32b_x16(tS + p_column(BIAS) + 16 * c, zero);
  tmem_st_32x32b_x16(tS + p_column(BIAS) + 16 * piece, p);
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
// sum of a flag over the 256 softmax threads: a barrier and a vote in one, so
// that all of them leave together
__device__ __forceinline__ bool any_of_softmax(bool x) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

// Bits of columns that hold +inf, -inf or NaN, and the sum of those values in one.
struct Kinds {
  uint32_t pos, neg, nan;
  __device__ __forceinline__ uint32_t any() const { return pos | neg | nan; }
  __device__ __forceinline__ uint32_t undefined() const { return nan | (pos & neg); }  // the sum is NaN
  __device__ __forceinline__ float sum(int e) const {
    return undefined() >> e & 1 ? NAN : pos >> e & 1 ? INFINITY : neg >> e & 1 ? -INFINITY : 0.f;
  }
};
// adds those of the 8 in x to k
template <int FMT>
__device__ __forceinline__ void find_kinds(const uint4& x, Kinds& k) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t h = w[e >> 1] >> (16 * (e & 1)) & 0xffffu;
    if (!not_finite16<FMT>(h)) continue;
    constexpr uint32_t frac = FMT == kF16 ? 0x03ffu : 0x007fu;
    (h & frac ? k.nan : h & 0x8000u ? k.neg : k.pos) |= 1u << e;
  }
}
// 4-D tensor map coordinates: (d, s, h, b)
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int d, int s, int h, int b,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(d), "r"(s), "r"(h), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

}  // namespace fa

// dims (d, s, h, b), element strides (b, h, s); box = one swizzle row
// (box_d elements = 128 bytes) x 128 rows.
// mn_major_tf32: the 128-byte swizzle with 32-byte atomicity that the MMA's
// MN-major tf32 operand layout (SWIZZLE_128B_BASE32B) expects (V of the tf32 path).
static bool make_tmap_4d(CUtensorMap* map, const void* base, int dtype, int64_t D, int64_t S, int64_t H, int64_t B,
                         const int64_t* strides_elems, bool mn_major_tf32 = false) {
  // dims (d, s, h, b); strides in bytes for s, h, b
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return false;
    fn = reinterpret_cast<EncodeFn>(p);
  }
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  const cuuint64_t es = dtype == B2_F32 ? 4 : 2;
  const cuuint64_t strides[3] = {(cuuint64_t)strides_elems[2] * es, (cuuint64_t)strides_elems[1] * es,
                                 (cuuint64_t)strides_elems[0] * es};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / es), 128, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == B2_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype == B2_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(map, dt, 4, const_cast<void*>(base),
            dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            mn_major_tf32 ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// element strides whose byte values are multiples of 16 (TMA)
static bool strides_ok(const int64_t* s, int dtype) {
  const int64_t m = dtype == B2_F32 ? 4 : 8;
  return s[0] % m == 0 && s[1] % m == 0 && s[2] % m == 0;
}

}  // namespace b2
