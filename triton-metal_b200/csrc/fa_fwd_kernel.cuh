// The tcgen05 prefill kernel (fa_fwd_sm100.cu: plain, causal and sliding-window
// attention; fa_scored_sm100.cu: documents, prefixes, capped and biased scores).
#pragma once
#include "attn_common.cuh"
#include "fa_common.cuh"
#include <limits.h>

namespace b2 {
namespace fa {

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
  static constexpr size_t kSmem = (size_t)kTile * (2 + kKStages + kVStages) + 1024 + 512;
  static_assert(HD % AE == 0, "head dim must fill whole swizzle rows");
};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.f;  // log2 units

struct Params {
  int B, Hq, Hkv, Sq, Skv, causal, q_tiles;
  int window;  // > 0 (causal only): key kv visible to qpos iff qpos - window < kv <= qpos
  int single;  // 1: one Q tile per CTA instead of a pair (small grids)
  float scale_log2;
  void* o;
  int64_t os_b, os_h, os_s;
  unsigned* err;
  // score forms and row ranges (SC kernels only)
  attn::RangeMask range;
  const float* slopes;     // [Hq] or null
  float cap_in, cap_log2;  // 2 log2 e scale / softcap; softcap * log2 e
  const uint16_t* v;       // V again, for values that are not finite
  int64_t vs_b, vs_h, vs_s;
};

// 4-D tensor map coordinates: (d, s, h, b)
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int d, int s, int h, int b,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(d), "r"(s), "r"(h), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

// ---------------------------------------------------------------------------
// Fast path v2: two Q tiles per CTA (ping-pong), P kept in TMEM.
//   TMEM (512 columns): tile u in {0, 1}: S_u / P_u at columns 256u, O_u at
//   256u + 128.  P_u (bf16, two per 32-bit column) overwrites the first 64
//   columns of S_u and is read by the TMEM-A form of tcgen05.mma.
//   MMA issue order per KV block j:  PV_0(j), S_0(j+1), PV_1(j), S_1(j+1),
//   so the tensor core works on one tile while the other tile's softmax
//   warpgroup runs.  MMAs from the single issuing thread execute in order,
//   which orders S_u(j+1) after PV_u(j) (both use the S/P columns) and makes
//   O_u quiescent whenever S_u(j) is complete.
//   warps: 0 TMA, 1 TMEM owner + MMA issuer, 4-7 softmax tile 0,
//          8-11 softmax tile 1 (warp w reads TMEM lanes 32 (w % 4) ..).
// ---------------------------------------------------------------------------
constexpr int kThreads2 = 384;

__device__ __forceinline__ bool key_masked(int kv, int qpos, const Params& p) {
  return kv >= p.Skv || (p.causal && kv > qpos) || (p.window > 0 && kv <= qpos - p.window);
}

// Row max of the raw S row (this thread's TMEM lane), masked keys -> -inf.
template <bool MASK>
__device__ __forceinline__ float row_max(uint32_t tS, int kv0, int qpos, const Params& p) {
  float mx = -INFINITY;
  // two 32-column loads per wait: 64 columns in flight
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    uint32_t sv[64];
    tc::tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
    tc::tmem_ld_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
    tc::tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
      float v0 = __uint_as_float(sv[e]), v1 = __uint_as_float(sv[e + 1]);
      if constexpr (MASK) {
        const int kv = kv0 + 32 * c + e;
        if (key_masked(kv, qpos, p)) v0 = -INFINITY;
        if (key_masked(kv + 1, qpos, p)) v1 = -INFINITY;
      }
      mx = max3(mx, v0, v1);
    }
  }
  return mx;
}

// p = exp2(s * scale_log2 - m) written over the S columns (P for the TMEM-A
// MMA): 16-bit pairs, or fp32 for the tf32 path; returns the row sum of p
// (two partial sums, even and odd keys, in one register pair).
template <bool MASK, int FMT>
__device__ __forceinline__ float exp_to_p(uint32_t tS, int kv0, int qpos, float mref, const Params& p) {
  uint64_t rs = 0;
  const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nm2 = f2_pack(-mref, -mref);
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    uint32_t sv[64];
    tc::tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
    tc::tmem_ld_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
    tc::tmem_ld_wait();
    uint32_t pk[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const uint64_t x = fma_f2((uint64_t)sv[2 * e] | ((uint64_t)sv[2 * e + 1] << 32), sc2, nm2);
      float p0, p1;
      // ~1/3 of the pairs on the FMA pipe (measured at C3: 1/4 and 1/3 both
      // ~1020 TF/s, 3/8 ~1005, 1/2 ~965; all-MUFU ~970)
      if (FMT != kTF32 && e % 3 == 2) {
        const uint64_t y = exp2_poly_f2(x);
        p0 = f2_lo(y);
        p1 = f2_hi(y);
      } else {
        p0 = ex2(f2_lo(x));
        p1 = ex2(f2_hi(x));
      }
      if constexpr (MASK) {
        const int kv = kv0 + 32 * c + 2 * e;
        if (key_masked(kv, qpos, p)) p0 = 0.f;
        if (key_masked(kv + 1, qpos, p)) p1 = 0.f;
      }
      rs = add_f2(rs, f2_pack(p0, p1));
      if constexpr (FMT == kF16) {
        __half2 hv = __floats2half2_rn(p0, p1);
        pk[e] = *reinterpret_cast<uint32_t*>(&hv);
      } else if constexpr (FMT == kBF16) {
        __nv_bfloat162 hv = __floats2bfloat162_rn(p0, p1);
        pk[e] = *reinterpret_cast<uint32_t*>(&hv);
      } else {
        sv[2 * e] = __float_as_uint(p0);
        sv[2 * e + 1] = __float_as_uint(p1);
      }
    }
    if constexpr (FMT == kTF32) {
      tmem_st_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sv));
      tmem_st_32x32b_x32(tS + 32 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
    } else {
      tmem_st_32x32b_x32(tS + 16 * c, pk);
    }
  }
  return f2_lo(rs) + f2_hi(rs);
}

// Bits of the keys of [lo, hi) among the 128 from kv0 on.
__device__ __forceinline__ void range_bits(uint32_t (&vis)[4], int lo, int hi, int kv0) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int a = min(max(lo - kv0 - 32 * w, 0), 32), z = min(max(hi - kv0 - 32 * w, 0), 32);
    const uint32_t below_z = z == 32 ? 0xffffffffu : (1u << z) - 1, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1;
    vis[w] = below_z & ~below_a;
  }
}

// SC: key ranges per row (documents, prefixes) and score forms, CAP: scores
// capped by a tanh, BIAS: minus slope times distance.  A tile in which some row
// must not see some key is "masked" there: its softmax takes a bit per key, and
// warps 2-3 go through its V tile first (they hand every V tile on) and zero
// what is infinite or NaN, since a weight of 0 would make NaN of it; rows that
// do see such a value get it added at the end.
template <int HD, int FMT, bool SC, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads2, 1)
fa_fwd2_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const Params p) {
  using Cf = FaCfg<HD, FMT>;
  constexpr int kTile = Cf::kTile, kAtom = Cf::kAtom;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* sQ = smem;                      // 2 tiles
  uint8_t* sK = sQ + 2 * kTile;
  uint8_t* sV = sK + kKStages * kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kVStages * kTile);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v_full = k_empty + kKStages;
  uint64_t* v_empty = v_full + kVStages;
  uint64_t* s_full = v_empty + kVStages;  // [2] per tile
  uint64_t* p_ready = s_full + 2;         // [2]
  uint64_t* o_done = p_ready + 2;         // [2]
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // SC only: a cleaned V tile per stage, row ranges of the softmax warps, a V
  // value that is not finite
  uint64_t* v_clean = reinterpret_cast<uint64_t*>(tmem_holder + 2);
  int4* s_range = reinterpret_cast<int4*>(bars + 24);
  volatile int* s_bad = reinterpret_cast<volatile int*>(s_range + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // one unit = a pair of Q tiles, or one Q tile when the grid would not fill
  // the SMs (p.single: the second softmax warpgroup idles, the CTAs halve)
  const int per = p.single ? 1 : 2;
  const int nunits = (p.q_tiles + per - 1) / per;
  const int pi = nunits - 1 - (int)blockIdx.x;  // longest causal units first
  const int h = blockIdx.y, b = blockIdx.z;
  const int hk = h / (p.Hq / p.Hkv);
  const int nkv_all = (p.Skv + BKV - 1) / BKV;
  // Tile u visits KV tiles kb[u] .. nkv[u]-1 (kb > 0 only with a sliding
  // window); the pair shares the K/V ring over the union jb .. nkv_max-1.
  int q0[2], nkv[2], kb[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    q0[u] = (per * pi + u) * BQ;
    nkv[u] = (u < per && per * pi + u < p.q_tiles)
                 ? (p.causal ? min(nkv_all, (q0[u] + BQ - 1) / BKV + 1) : nkv_all)
                 : 0;
    kb[u] = p.window > 0 ? min(max(0, q0[u] - p.window + 1) / BKV, nkv[u]) : 0;
  }
  int nkv_max = max(nkv[0], nkv[1]);
  int jb = kb[0];
  int lo_most[2] = {0, 0}, hi_least[2] = {INT_MAX, INT_MAX};  // SC: keys every row of a tile sees
  auto active = [&](int u, int j) { return j >= kb[u] && j < nkv[u]; };
  // SC: some row of tile u must not see some key of KV tile j
  auto masked = [&](int u, int j) { return j * BKV < lo_most[u] || j * BKV + BKV > hi_least[u]; };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&s_full[u], 1);
      mbar_init(&p_ready[u], 4);
      mbar_init(&o_done[u], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    if constexpr (SC) {
      for (int i = 0; i < kVStages; ++i) mbar_init(&v_clean[i], 64);
      *s_bad = 0;
    }
    fence_mbar_init();
  }
  int row_lo = 0, row_hi = 0;  // SC: keys of this softmax thread's row
  if constexpr (SC) {
    if (warp >= 4) {
      const int u = (warp - 4) >> 2, row = q0[u] + (warp & 3) * 32 + lane;
      const bool exists = nkv[u] > 0 && row < p.Sq;
      if (exists) attn::row_range(p.range, b, row, p.Skv, row_lo, row_hi);
      const bool sees = row_hi > row_lo;
      // smallest / largest first key, largest / smallest end; a row that sees
      // nothing makes every tile a masked one
      int4 v = make_int4(sees ? row_lo : INT_MAX, exists ? (sees ? row_lo : INT_MAX) : 0, sees ? row_hi : 0,
                         exists ? (sees ? row_hi : 0) : INT_MAX);
      v.x = __reduce_min_sync(0xffffffffu, v.x);
      v.y = __reduce_max_sync(0xffffffffu, v.y);
      v.z = __reduce_max_sync(0xffffffffu, v.z);
      v.w = __reduce_min_sync(0xffffffffu, v.w);
      if (lane == 0) s_range[warp - 4] = v;
    }
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_holder, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  if constexpr (SC) {
    // KV tiles from the first key that a row of the tile sees to the last.  A
    // row that sees anything sees itself or everything, so the two tiles' spans
    // touch and the pair's union has no gap.
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int lo = INT_MAX, hi = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int4 v = s_range[4 * u + w];
        lo = min(lo, v.x);
        lo_most[u] = max(lo_most[u], v.y);
        hi = max(hi, v.z);
        hi_least[u] = min(hi_least[u], v.w);
      }
      kb[u] = hi > 0 ? lo / BKV : 0;
      nkv[u] = (hi + BKV - 1) / BKV;
    }
    nkv_max = max(nkv[0], nkv[1]);
    jb = nkv[0] == 0 ? kb[1] : nkv[1] == 0 ? kb[0] : min(kb[0], kb[1]);
  }

  if (warp == 0) {
    // ---------------------------------- TMA ----------------------------------
    if (lane == 0) {
      const int ntiles = nkv[1] > 0 ? 2 : 1;
      mbar_arrive_expect_tx(q_full, ntiles * kTile);
      for (int u = 0; u < ntiles; ++u)
#pragma unroll
        for (int a = 0; a < Cf::NATOM; ++a) tma_load_4d(sQ + u * kTile + a * kAtom, &tmQ, a * Cf::AE, q0[u], h, b, q_full);
      int kst = 0, vst = 0;
      uint32_t kph = 0, vph = 0;
      for (int j = jb; j < nkv_max; ++j) {
        if (!wait_abort(&k_empty[kst], kph ^ 1, p.err, 0xB2300001u, abort_flag)) break;
        mbar_arrive_expect_tx(&k_full[kst], kTile);
#pragma unroll
        for (int a = 0; a < Cf::NATOM; ++a)
          tma_load_4d(sK + kst * kTile + a * kAtom, &tmK, a * Cf::AE, j * BKV, hk, b, &k_full[kst]);
        if (!wait_abort(&v_empty[vst], vph ^ 1, p.err, 0xB2300002u, abort_flag)) break;
        mbar_arrive_expect_tx(&v_full[vst], kTile);
#pragma unroll
        for (int a = 0; a < Cf::NATOM; ++a)
          tma_load_4d(sV + vst * kTile + a * kAtom, &tmV, a * Cf::AE, j * BKV, hk, b, &v_full[vst]);
        if (++kst == kKStages) { kst = 0; kph ^= 1; }
        if (++vst == kVStages) { vst = 0; vph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------- MMA ----------------------------------
    if (lane == 0) {
      constexpr uint32_t idS = idesc_fmt(BQ, BKV, FMT, false);
      constexpr uint32_t idPV = idesc_fmt(BQ, HD, FMT, true);
      bool ok = wait_abort(q_full, 0, p.err, 0xB2300003u, abort_flag);
      int kst = 0, vst = 0;
      uint32_t kph = 0, vph = 0;
      auto issue_s = [&](int u) {
#pragma unroll
        for (int kk = 0; kk < HD / Cf::KSTEP; ++kk) {
          const uint64_t da = tc::desc_kmajor_sw128(sQ + u * kTile + (kk >> 2) * kAtom + (kk & 3) * 32);
          const uint64_t db = tc::desc_kmajor_sw128(sK + kst * kTile + (kk >> 2) * kAtom + (kk & 3) * 32);
          mma_ss<FMT>(tmem + 256 * u, da, db, idS, kk != 0);
        }
        tc::commit(&s_full[u]);
      };
      // prologue: S_u(0)
      if (ok && nkv_max > jb) {
        ok = wait_abort(&k_full[kst], kph, p.err, 0xB2300004u, abort_flag);
        if (ok) {
          tc::fence_after_sync();
          for (int u = 0; u < 2; ++u)
            if (active(u, jb)) issue_s(u);
          tc::commit(&k_empty[kst]);
          if (++kst == kKStages) { kst = 0; kph ^= 1; }
        }
      }
      for (int j = jb; j < nkv_max && ok; ++j) {
        if (!wait_abort(SC ? &v_clean[vst] : &v_full[vst], vph, p.err, 0xB2300005u, abort_flag)) {
          ok = false;
          break;
        }
        const bool next_k = active(0, j + 1) || active(1, j + 1);
        bool k_waited = false;
        for (int u = 0; u < 2 && ok; ++u) {
          if (active(u, j)) {
            if (!wait_abort(&p_ready[u], (j - kb[u]) & 1, p.err, 0xB2300006u, abort_flag)) {
              ok = false;
              break;
            }
            tc::fence_after_sync();
#pragma unroll
            // one k-step = KSTEP keys: KSTEP rows of V, 8 TMEM columns of P.
            // V is the MN-major B operand: 128-byte rows along d, atoms of
            // 8 rows (16-bit, 128B swizzle) or of 4 rows (tf32, 128B swizzle
            // with 32-byte atomicity, descriptor layout 1) stacked along K.
            for (int kk = 0; kk < BKV / Cf::KSTEP; ++kk) {
              const uint64_t db =
                  FMT == kTF32 ? tc::smem_desc(sV + vst * kTile + kk * Cf::KSTEP * 128, kAtom, 512, 1)
                               : tc::smem_desc(sV + vst * kTile + kk * Cf::KSTEP * 128, kAtom, 1024, tc::kSwizzle128B);
              mma_ts<FMT>(tmem + 256 * u + 128, tmem + 256 * u + kk * 8, db, idPV, (j != kb[u]) || kk != 0);
            }
            if (j == nkv[u] - 1) tc::commit(&o_done[u]);
          }
          if (active(u, j + 1)) {
            if (!k_waited) {
              if (!wait_abort(&k_full[kst], kph, p.err, 0xB2300007u, abort_flag)) {
                ok = false;
                break;
              }
              tc::fence_after_sync();
              k_waited = true;
            }
            issue_s(u);
          }
        }
        if (!ok) break;
        tc::commit(&v_empty[vst]);
        if (++vst == kVStages) { vst = 0; vph ^= 1; }
        if (next_k) {
          tc::commit(&k_empty[kst]);
          if (++kst == kKStages) { kst = 0; kph ^= 1; }
        }
      }
      if (!ok) {
        tc::commit(drain);
        mbar_wait(drain, 0, p.err, 0xB2300008u);
      }
    }
  } else if (warp < 4) {
    // ------------------------- V of masked tiles (SC) -------------------------
    if constexpr (SC) {
      int vst = 0;
      uint32_t vph = 0;
      const int t = threadIdx.x - 64;
      for (int j = jb; j < nkv_max; ++j) {
        // every tile passes through here, so that these warps are never a ring
        // turn behind a stage (a parity wait cannot tell that)
        if (!wait_abort(&v_full[vst], vph, p.err, 0xB230000Bu, abort_flag)) break;
        if ((active(0, j) && masked(0, j)) || (active(1, j) && masked(1, j))) {
          uint4* tile = reinterpret_cast<uint4*>(sV + vst * kTile);
          bool bad = false;
#pragma unroll 8
          for (int i = t; i < kTile / 16; i += 64) {
            uint4 x = tile[i];
            if (zero_not_finite<FMT>(x)) {
              tile[i] = x;
              bad = true;
            }
          }
          if (bad) *s_bad = 1;
          tc::fence_proxy_async_smem();
        }
        mbar_arrive(&v_clean[vst]);
        if (++vst == kVStages) { vst = 0; vph ^= 1; }
      }
    }
  } else {
    // -------------------------------- softmax --------------------------------
    const int u = (warp - 4) >> 2;
    const int qw = warp & 3;
    const int r = qw * 32 + lane;
    const int qpos = q0[u] + r;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const uint32_t tS = tmem + 256 * u + lane_off, tO = tS + 128;
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    Score score = {p.scale_log2, 0.f, 0.f, 0.f, 0.f};
    if constexpr (CAP) {
      score.cap_in = p.cap_in;
      score.cap_log2 = p.cap_log2;
    }
    float slope = 0.f;
    if constexpr (BIAS) slope = p.slopes[h] * kLog2e;
    for (int j = kb[u]; j < nkv[u] && ok; ++j) {
      if (!wait_abort(&s_full[u], (j - kb[u]) & 1, p.err, 0xB2300009u, abort_flag)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      const int kv0 = j * BKV;
      bool need_mask;
      uint32_t vis[4] = {0, 0, 0, 0};
      float mx;
      if constexpr (SC) {
        need_mask = masked(u, j);
        if constexpr (BIAS) {
          // the bias is linear over the tile unless the tile's rows lie in it
          const bool before = kv0 + BKV - 1 <= q0[u], behind = kv0 >= q0[u] + BQ - 1;
          need_mask = need_mask || !(before || behind);
          score.dist = (float)(qpos - kv0);
          score.slope = need_mask || before ? slope : -slope;
        }
        if (need_mask) range_bits(vis, row_lo, row_hi, kv0);
        mx = need_mask ? score_max<true, CAP, BIAS>(tS, vis, score) : score_max<false, CAP, BIAS>(tS, vis, score);
      } else {
        need_mask = (p.causal && kv0 + BKV - 1 > q0[u]) || kv0 + BKV > p.Skv ||
                    (p.window > 0 && kv0 <= q0[u] + BQ - 1 - p.window);
        // pass 1: row max of the raw scores (scale > 0 commutes with max)
        mx = need_mask ? row_max<true>(tS, kv0, qpos, p) : row_max<false>(tS, kv0, qpos, p);
        mx *= p.scale_log2;
      }
      // lazy, warp-uniform rescale of O (O_u is quiescent: PV_u(j-1) finished)
      const bool need = mx > m_used + kRescaleThreshold;
      const float alpha = need ? ((m_used == -INFINITY) ? 0.f : ex2(m_used - mx)) : 1.f;
      if (need) {
        l *= alpha;
        m_used = mx;
      }
      if (__any_sync(0xffffffffu, need) && j > kb[u]) {
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
      // pass 2: p = exp2(s * scale - m) -> bf16 pairs over the S columns already read
      const float mref = (m_used == -INFINITY) ? 0.f : m_used;
      float rs;
      if constexpr (SC)
        rs = need_mask ? score_exp<true, FMT, CAP, BIAS>(tS, vis, mref, score)
                       : score_exp<false, FMT, CAP, BIAS>(tS, vis, mref, score);
      else
        rs = need_mask ? exp_to_p<true, FMT>(tS, kv0, qpos, mref, p)
                       : exp_to_p<false, FMT>(tS, kv0, qpos, mref, p);
      l += rs;
      tmem_st_wait();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[u]);
    }
    if constexpr (SC) {
      // no row of the tile sees anything: zeros
      if (nkv[u] == 0 && (u < per) && qpos < p.Sq) {
        uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.o) + b * p.os_b + h * p.os_h +
                                              (int64_t)qpos * p.os_s);
        for (int e = 0; e < HD / 8; ++e) dst[e] = make_uint4(0, 0, 0, 0);
      }
    }
    // epilogue: O_u / l -> global (rows beyond Sq are not stored)
    if (ok && nkv[u] > kb[u] && wait_abort(&o_done[u], 0, p.err, 0xB230000Au, abort_flag)) {
      tc::fence_after_sync();
      const float inv = l > 0.f || (SC && l != l) ? 1.f / l : 0.f;
      const int64_t orow = b * p.os_b + h * p.os_h + (int64_t)qpos * p.os_s;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tc::tmem_ld_32x32b_x32(tO + 32 * c, o);
        tc::tmem_ld_wait();
        if constexpr (SC) {
          if (*s_bad) {
            for (int key = row_lo; key < row_hi; ++key) {
              const uint16_t* v = p.v + b * p.vs_b + hk * p.vs_h + (int64_t)key * p.vs_s + 32 * c;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const uint16_t x = v[e];
                if (not_finite16<FMT>(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + widen16<FMT>(x));
              }
            }
          }
          if (l == 0.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
        }
        if (qpos < p.Sq) {
          if constexpr (FMT == kTF32) {
            float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.o) + orow + 32 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[e] = make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                   __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
          } else {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float a = __uint_as_float(o[2 * e]) * inv, bb = __uint_as_float(o[2 * e + 1]) * inv;
              if constexpr (FMT == kF16) {
                __half2 hv = __floats2half2_rn(a, bb);
                pk[e] = *reinterpret_cast<uint32_t*>(&hv);
              } else {
                __nv_bfloat162 hv = __floats2bfloat162_rn(a, bb);
                pk[e] = *reinterpret_cast<uint32_t*>(&hv);
              }
            }
            uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.o) + orow + 32 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[e] = make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
          }
        }
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
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
