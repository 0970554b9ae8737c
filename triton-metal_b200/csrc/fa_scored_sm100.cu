// FlashAttention forward with document and prefix masks, capped scores and a
// distance bias: key ranges per row and score forms, on tcgen05 here (16-bit,
// head dim 64 / 128) and on the CUDA cores in attn_simt.cu (the rest, fp32
// arithmetic).  The reference has causal masking only
// (_msl_templates.py:1610-1619).
//
//   s = scale q.k;  softcap: s = softcap tanh(s / softcap);  s -= slope |i - j|
//
// Every mask is one key range per query row (attn::row_range), so a Q tile
// visits the KV tiles from its rows' first visible key to their last, and only
// tiles at the ranges' ends are masked.  Capped and biased scores cost softmax
// issue slots, not memory.
#include "attn_common.cuh"
#include "fa_common.cuh"
#include <limits.h>
#include <math.h>

namespace b2 {
namespace scored {

using namespace fa;

// ---------------------------------------------------------------------------
// The pipeline of the plain prefill kernel (fa_fwd_sm100.cu: two Q tiles in
// ping-pong, P in TMEM), made persistent: with short documents a unit (a pair
// of Q tiles of one head) has a handful of KV tiles, and what counts is how
// soon the next one starts.  One CTA per SM walks units; the next unit's first
// Q, K and V tiles are loaded and its first S is computed while this one's last
// softmax and output are under way (three Q tiles of room and two K tiles,
// where the plain kernel has two and three).
//   warp 0      TMA
//   warp 1      TMEM owner, MMA issuer
//   warps 2-3   key ranges of the next unit: which KV tiles its Q tiles visit,
//               which of them are masked
//   warps 4-11  two softmax warpgroups, one per Q tile, one row per thread
// Measured: 2 x 8192 tokens in 11 documents a row, causal, 32 / 8 heads of 128,
// bf16: 274 to 282 us, 430 TF/s of visible pairs (one document of 8192 in each of 4
// rows: 950, where the plain kernel has 1040);
// 6001 tokens, causal, cap 50, 16 / 8 heads, fp16: 275 us, 540 TF/s of visible
// pairs; 3 x 1111 tokens, prefix 300 and bias, 12 heads of 64: 40 us.  In the
// capped case the tensor pipe is active for 28 % of the cycles and the softmax
// warps, two a scheduler, issue in 42 %: their chains of dependent instructions
// set the time, and more warps of them do not fit the registers.
// ---------------------------------------------------------------------------
constexpr int kThreads = 384;
constexpr int kQ = 3, kK = 2, kV = 2;  // tiles of each ring

struct Params {
  int B, Hq, Hkv, Sq, Skv, q_tiles;
  int per, n_units;        // Q tiles of a unit (1 where pairs would not fill the SMs); units of a head
  attn::RangeMask range;
  Cap cap;
  const float* slopes;     // [Hq]
  void* o;
  int64_t os_b, os_h, os_s;
  const uint16_t *q, *k, *v;  // for rows that are looked at again
  int64_t qs[3], ks[3], vs[3];
  unsigned* err;
};

// Unit of a CTA's turn: the rows furthest back first (causal rows: the longest),
// heads of one kv head next to one another (their K/V stays in L2), turns in
// alternating direction so that nobody gets the longest of each.
struct Unit {
  int b, h, q0;  // q0: first row
};
__device__ __forceinline__ bool unit_of(const Params& p, int turn, Unit& u) {
  const int64_t G = gridDim.x, n = (int64_t)p.n_units * p.Hq * p.B;
  const int64_t at = turn * G + (turn & 1 ? G - 1 - blockIdx.x : blockIdx.x);
  if (at >= n) return false;
  const uint32_t heads = (uint32_t)p.Hq * p.B, x = (uint32_t)at;
  const uint32_t row = x / heads, bh = x - row * heads;
  u.b = bh / (uint32_t)p.Hq;
  u.h = bh - u.b * p.Hq;
  u.q0 = (p.n_units - 1 - (int)row) * p.per * BQ;
  return true;
}

// What warps 2-3 find out about a unit's two Q tiles.  KV tiles are counted in
// the order in which they are taken: from the first key on, or with a bias from
// the last one back (tile number -j, so that all the loops count up).
struct Info {
  bool has[2];                  // a row of the tile sees anything
  int kb[2], nkv[2];            // turns kb .. nkv - 1
  int lo_most[2], hi_least[2];  // keys that every row of the tile sees
  __device__ __forceinline__ bool active(int u, int j) const { return j >= kb[u] && j < nkv[u]; }
  __device__ __forceinline__ bool masked(int u, int tile) const {
    return tile * BKV < lo_most[u] || tile * BKV + BKV > hi_least[u];
  }
  __device__ __forceinline__ bool any() const { return has[0] || has[1]; }
  __device__ __forceinline__ int first() const { return !has[0] ? kb[1] : !has[1] ? kb[0] : min(kb[0], kb[1]); }
  __device__ __forceinline__ int last() const { return !has[0] ? nkv[1] : !has[1] ? nkv[0] : max(nkv[0], nkv[1]); }
  // the Q tile whose turn comes first
  __device__ __forceinline__ int lead() const { return !has[0] || (has[1] && kb[1] < kb[0]) ? 1 : 0; }
};

// Bits of the keys of [lo, hi) among the 128 from kv0 on.
__device__ __forceinline__ void range_bits(uint32_t (&vis)[4], int lo, int hi, int kv0) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int a = min(max(lo - kv0 - 32 * w, 0), 32), z = min(max(hi - kv0 - 32 * w, 0), 32);
    const uint32_t below_z = z == 32 ? 0xffffffffu : (1u << z) - 1, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1;
    vis[w] = below_z & ~below_a;
  }
}

// Rows looked at again.  A tile's PV takes every key of the tile, and a hidden one's
// infinity or NaN in V times its weight of 0 is NaN.  In fp16 a visible one's weight
// may round to 0 as well (below 2^-25, where bf16's last is fp32's), which makes NaN
// of an infinity.  So rows whose output is not finite are looked at once more when
// all turns are over (no wait with a limit is left then, and the tiles' shared
// memory is free):
//   * a key in V that is not finite and hidden from a row (fp16: from any of the
//     warp's 32 rows) in a tile that was taken for it: the row is computed anew over
//     the keys that it sees, 32 at a time, one key a lane for the scores and HD / 32
//     columns a lane for PV;
//   * fp16, such keys only where all rows see them: their columns are the sum of
//     those values, whatever the weights;
//   * else the row is what the formula gives.
// Each softmax warp finds out about its own rows; rows to compute anew go through a
// list in shared memory to all eight, four at a time.  8192 tokens, causal, 32 heads
// of 128: 0.57 ms clean, 0.64 (fp16 0.75) with a NaN in V of token 0, which all rows
// see, 3.1 with NaN in 96 tokens of padding, whose tile 32 rows of each head share.
template <int FMT>
__device__ __forceinline__ bool any_not_finite(const uint4& x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool hit = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) hit |= not_finite16<FMT>(w[e]) | not_finite16<FMT>(w[e] >> 16);
  return hit;
}

// First (LAST: last) of the keys [a, z) with a value in V (rows vs apart) that is
// not finite; LAST ? -1 : INT_MAX where there is none.  For a whole warp.
template <int HD, int FMT, bool LAST>
__device__ __forceinline__ int bad_key(const uint16_t* v, int64_t vs, int a, int z) {
  constexpr int NL = HD / 8, KEYS = 32 / NL, U = 4;  // lanes a key, keys side by side, steps in flight
  const int lane = threadIdx.x & 31, none = LAST ? -1 : INT_MAX;
  for (int i0 = 0; i0 < z - a; i0 += KEYS * U) {
    uint4 x[U];
    int best = none;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int i = i0 + e * KEYS + lane / NL, key = LAST ? z - 1 - i : a + i;
      x[e] = i < z - a ? *reinterpret_cast<const uint4*>(v + key * vs + lane % NL * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int i = i0 + e * KEYS + lane / NL, key = LAST ? z - 1 - i : a + i;
      if (any_not_finite<FMT>(x[e])) best = LAST ? max(best, key) : min(best, key);
    }
    best = LAST ? __reduce_max_sync(0xffffffffu, best) : __reduce_min_sync(0xffffffffu, best);
    if (best != none) return best;
  }
  return none;
}

// HD / 32 columns of V, this lane's
template <int HD, int FMT>
__device__ __forceinline__ void load_columns(float (&o)[HD / 32], const uint16_t* v) {
  const int lane = threadIdx.x & 31;
  uint32_t w[HD / 64];
  if constexpr (HD == 128) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(v + 4 * lane);
  else w[0] = *reinterpret_cast<const uint32_t*>(v + 2 * lane);
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) {
    o[2 * e] = widen16<FMT>((uint16_t)w[e]);
    o[2 * e + 1] = widen16<FMT>((uint16_t)(w[e] >> 16));
  }
}

// Whether V of the keys lo and hi - 1, the first and the last that a row sees, makes
// NaN of all its columns (as in a prompt that is NaN from some token on).
template <int HD, int FMT>
__device__ __forceinline__ bool all_nan(const uint16_t* vb, int64_t vs, int lo, int hi) {
  float x[HD / 32], y[HD / 32];
  load_columns<HD, FMT>(x, vb + lo * vs);
  load_columns<HD, FMT>(y, vb + (hi - 1) * vs);
  bool nan = true;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) nan = nan && (x[e] != x[e] || y[e] != y[e]);
  return __all_sync(0xffffffffu, nan);
}

// The rows first + r, r in `rows` (a bit each, kAgain at most), of a unit over the
// keys that they see, by one warp; they share what they load.
constexpr int kAgain = 4;
template <int HD, int FMT, bool CAP, bool BIAS>
__device__ __forceinline__ void compute_rows(const Params& p, const Unit& un, int first, uint32_t rows, const Score& sc) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31, hk = un.h / (p.Hq / p.Hkv);
  const uint16_t* qb = p.q + un.b * p.qs[0] + un.h * p.qs[1];
  const uint16_t* kb = p.k + un.b * p.ks[0] + hk * p.ks[1];
  const uint16_t* vb = p.v + un.b * p.vs[0] + hk * p.vs[1];
  int row[kAgain], from[kAgain], to[kAgain], a = INT_MAX, z = 0;  // row < 0: none
#pragma unroll
  for (int i = 0; i < kAgain; ++i) {
    row[i] = rows ? first + __ffs(rows) - 1 : -1;
    from[i] = to[i] = 0;
    if (rows) {
      attn::row_range(p.range, un.b, row[i], p.Skv, from[i], to[i]);
      a = min(a, from[i]);
      z = max(z, to[i]);
    }
    rows &= rows - 1;
  }
  float m[kAgain], l[kAgain], acc[kAgain][V];
#pragma unroll
  for (int i = 0; i < kAgain; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[i][e] = 0.f;
  }
  for (int key0 = a; key0 < z; key0 += 32) {
    const int key = key0 + lane;
    float w[kAgain] = {};  // scores, then weights; < 0: the row does not see the key
    if (key < z) {
      const uint16_t* k = kb + key * p.ks[2];
#pragma unroll 4
      for (int d = 0; d < HD; d += 8) {
        const uint4 y = *reinterpret_cast<const uint4*>(k + d);
        const uint32_t b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < kAgain; ++i) {
          const uint4 q = *reinterpret_cast<const uint4*>(qb + max(row[i], 0) * p.qs[2] + d);
          const uint32_t c[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[i] = fmaf(widen16<FMT>((uint16_t)c[e]), widen16<FMT>((uint16_t)b[e]), w[i]);
            w[i] = fmaf(widen16<FMT>((uint16_t)(c[e] >> 16)), widen16<FMT>((uint16_t)(b[e] >> 16)), w[i]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAgain; ++i) {
      const bool sees = key >= from[i] && key < to[i];
      float add = 0.f;
      if constexpr (BIAS) add = -sc.slope0 * fabsf((float)(row[i] - key));
      const float x = CAP ? capped_any(w[i], sc, add) : fmaf(w[i], sc.scale_log2, add);
      float mx = sees ? x : -INFINITY;
#pragma unroll
      for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float mn = fmaxf(m[i], mx), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = m[i] == -INFINITY ? 0.f : ex2(m[i] - ref);
      w[i] = sees ? ex2(x - ref) : -1.f;
      m[i] = mn;
      l[i] = l[i] * alpha + (sees ? w[i] : 0.f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[i][e] *= alpha;
    }
    const int n = min(z - key0, 32);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      float y[V];
      load_columns<HD, FMT>(y, vb + (key0 + j) * p.vs[2]);
#pragma unroll
      for (int i = 0; i < kAgain; ++i) {
        const float wj = __shfl_sync(0xffffffffu, w[i], j);
        if (!(wj < 0.f))
#pragma unroll
          for (int e = 0; e < V; ++e) acc[i][e] = fmaf(wj, y[e], acc[i][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kAgain; ++i) {
#pragma unroll
    for (int off = 16; off; off >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
    if (row[i] < 0) continue;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    uint16_t* o = reinterpret_cast<uint16_t*>(p.o) + un.b * p.os_b + un.h * p.os_h + row[i] * p.os_s + V * lane;
#pragma unroll
    for (int e = 0; e < V / 2; ++e)
      reinterpret_cast<uint32_t*>(o)[e] = narrow2<FMT>(acc[i][2 * e] * inv, acc[i][2 * e + 1] * inv);
  }
}

// fp16, 32 rows (sees: this lane's row) whose keys that are not finite in V are all
// among [a, z), which each of them sees.  Returns those of them to compute anew, a
// bit each.
template <int HD>
__device__ __forceinline__ uint32_t columns_again(const Params& p, const Unit& un, int first, bool sees, int a, int z,
                                                  const uint16_t* vb) {
  constexpr int NL = HD / 8, KEYS = 32 / NL, U = 8;
  const int lane = threadIdx.x & 31;
  const uint32_t rows = __ballot_sync(0xffffffffu, sees);
  auto at = [&](int r) {  // 8 columns of row first + r
    return reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.o) + un.b * p.os_b + un.h * p.os_h + (first + r) * p.os_s +
                                    lane % NL * 8);
  };
  uint32_t want = 0;  // this lane's columns, 8 (lane % NL) .., that are NaN in some row
  for (uint32_t left = rows; left; left &= left - 1) {
    Kinds have = {0, 0, 0};
    find_kinds<kF16>(*at(__ffs(left) - 1), have);
    want |= have.nan;
  }
  // V from key a on, until those columns are known to be NaN by the formula
  Kinds k = {0, 0, 0};
  for (int i0 = a; i0 < z; i0 += KEYS * U) {
    if (__all_sync(0xffffffffu, !(want & ~k.undefined()))) return 0;
    uint4 x[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int key = i0 + e * KEYS + lane / NL;
      x[e] = key < z ? *reinterpret_cast<const uint4*>(vb + key * p.vs[2] + lane % NL * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < U; ++e)
      if (any_not_finite<kF16>(x[e])) find_kinds<kF16>(x[e], k);
#pragma unroll
    for (int off = NL; off < 32; off <<= 1) {
      k.pos |= __shfl_xor_sync(0xffffffffu, k.pos, off);
      k.neg |= __shfl_xor_sync(0xffffffffu, k.neg, off);
      k.nan |= __shfl_xor_sync(0xffffffffu, k.nan, off);
    }
  }
  const uint32_t wrong = k.any() & ~k.undefined();
  uint32_t anew = 0;
  for (uint32_t left = rows; left; left &= left - 1) {
    const int r = __ffs(left) - 1;
    uint4 x = *at(r);
    Kinds have = {0, 0, 0};
    find_kinds<kF16>(x, have);
    if (__all_sync(0xffffffffu, have.nan == 0xffu)) {  // its scores, or all columns
      anew |= 1u << r;
      continue;
    }
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (have.nan & wrong & 1u << e) {
        const uint32_t h = __half_as_ushort(__float2half_rn(k.sum(e)));
        w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | h << 16 : (w[e >> 1] & 0xffff0000u) | h;
      }
    if (lane < NL && (have.nan & wrong)) *at(r) = x;
  }
  return anew;
}

// Which of the rows first .. first + 31 of the Q tile from row q0 on to compute
// anew, a bit each.
template <int HD, int FMT>
__device__ __forceinline__ uint32_t rows_again(const Params& p, const Unit& un, int q0, int first) {
  const int lane = threadIdx.x & 31, hk = un.h / (p.Hq / p.Hkv);
  const uint16_t* vb = p.v + un.b * p.vs[0] + hk * p.vs[1];
  int t0 = INT_MAX, t1 = 0, lo = 0, hi = 0;  // the tile's first key and end; this lane's row
  for (int i = 0; i < BQ / 32; ++i) {
    const int row = q0 + 32 * i + lane;
    int a = 0, z = 0;
    if (row < p.Sq) attn::row_range(p.range, un.b, row, p.Skv, a, z);
    if (z > a) t0 = min(t0, a), t1 = max(t1, z);
    if (q0 + 32 * i == first) lo = a, hi = z;
  }
  t0 = __reduce_min_sync(0xffffffffu, t0) / BKV * BKV;
  t1 = min((__reduce_max_sync(0xffffffffu, t1) + BKV - 1) / BKV * BKV, p.Skv);  // zeros behind the last key
  const bool sees = hi > lo;
  const int before = __reduce_max_sync(0xffffffffu, sees ? lo : 0);
  const int behind = __reduce_min_sync(0xffffffffu, sees ? hi : INT_MAX);
  const int bad0 = bad_key<HD, FMT, false>(vb, p.vs[2], t0, before);
  const int bad1 = bad_key<HD, FMT, true>(vb, p.vs[2], behind, t1);
  if (bad0 == INT_MAX && bad1 == -1) {
    if constexpr (FMT == kF16) return columns_again<HD>(p, un, first, sees, before, behind, vb);
    return 0;
  }
  uint32_t again = __ballot_sync(0xffffffffu, sees && (FMT == kF16 || bad0 < lo || bad1 >= hi));
  for (uint32_t left = again; left; left &= left - 1) {
    const int r = __ffs(left) - 1;
    if (all_nan<HD, FMT>(vb, p.vs[2], __shfl_sync(0xffffffffu, lo, r), __shfl_sync(0xffffffffu, hi, r))) again &= ~(1u << r);
  }
  return again;
}

template <int HD, int FMT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
scored_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
              const __grid_constant__ CUtensorMap tmV, const Params p) {
  using Cf = FaCfg<HD, FMT>;
  constexpr int kTile = Cf::kTile, kAtom = Cf::kAtom;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* sQ = smem;  // a unit's two Q tiles and the next one's first
  uint8_t* sK = sQ + kQ * kTile;
  uint8_t* sV = sK + kK * kTile;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sV + kV * kTile);
  uint64_t* q_empty = q_full + kQ;
  uint64_t* k_full = q_empty + kQ;
  uint64_t* k_empty = k_full + kK;
  uint64_t* v_full = k_empty + kK;
  uint64_t* v_empty = v_full + kV;
  uint64_t* s_full = v_empty + kV;            // [2] per Q tile
  uint64_t* p_ready = s_full + 2;             // [2]
  uint64_t* o_done = p_ready + 2;             // [2]
  uint64_t* info_full = o_done + 2;           // [2] by unit parity
  uint64_t* info_empty = info_full + 2;       // [2]
  uint64_t* drain = info_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int4* s_info = reinterpret_cast<int4*>(q_full + 32);                         // [2 parities][2 warps][2 tiles]
  static_assert(2 * kQ + 2 * kK + 2 * kV + 11 + 1 <= 32, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < kK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&s_full[u], 1);
      mbar_init(&p_ready[u], 4);
      mbar_init(&o_done[u], 1);
      mbar_init(&info_full[u], 64);
      mbar_init(&info_empty[u], 10);  // TMA, MMA, 8 softmax warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_holder, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_holder;

  auto tile_of = [](int j) { return BIAS ? -j : j; };  // KV tile of a turn
  // The info of turn k, once it is there; every reader says that it has it.
  auto read_info = [&](int k, Info& f) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int4 a = s_info[(k & 1) * 4 + u], b = s_info[(k & 1) * 4 + 2 + u];
      const int lo = min(a.x, b.x), hi = max(a.z, b.z);
      f.lo_most[u] = max(a.y, b.y);
      f.hi_least[u] = min(a.w, b.w);
      // A row that sees anything sees itself or everything, so the two tiles'
      // spans touch and the pair's union has no gap.
      f.has[u] = hi > 0;
      const int t0 = hi > 0 ? lo / BKV : 0, t1 = (hi + BKV - 1) / BKV;  // KV tiles t0 .. t1 - 1
      f.kb[u] = BIAS ? 1 - t1 : t0;
      f.nkv[u] = hi > 0 ? (BIAS ? 1 - t0 : t1) : f.kb[u];
    }
  };

  Unit un;
  Info f;
  if (warp == 0) {
    // ---------------------------------- TMA ----------------------------------
    if (lane == 0) {
      int kst = 0, vst = 0;
      uint32_t kph = 0, vph = 0, qn = 0;  // qn: Q tiles loaded
      bool ok = true;
      auto load = [&](const CUtensorMap* map, uint8_t* tile, uint64_t* bar, int row, int h, int b) {
        mbar_arrive_expect_tx(bar, kTile);
#pragma unroll
        for (int a = 0; a < Cf::NATOM; ++a) tma_load_4d(tile + a * kAtom, map, a * Cf::AE, row, h, b, bar);
      };
      auto load_q = [&](int u) {
        const uint32_t at = qn % kQ;
        ok = ok && wait_abort(&q_empty[at], ((qn / kQ) & 1) ^ 1, p.err, 0xB2600002u, abort_flag);
        if (ok) load(&tmQ, sQ + at * kTile, &q_full[at], un.q0 + u * BQ, un.h, un.b);
        ++qn;
      };
      for (int k = 0; ok && unit_of(p, k, un); ++k) {
        ok = wait_abort(&info_full[k & 1], (k >> 1) & 1, p.err, 0xB2600001u, abort_flag);
        if (!ok) break;
        read_info(k, f);
        mbar_arrive(&info_empty[k & 1]);
        const int jb = f.first(), je = f.last();
        if (!f.any()) continue;
        const int hk = un.h / (p.Hq / p.Hkv);
        // the unit's first Q tile has room while the unit before is still at
        // work; its second one takes the place of that unit's first
        const int u0 = f.lead();
        load_q(u0);
        for (int j = jb; j < je && ok; ++j) {
          ok = wait_abort(&k_empty[kst], kph ^ 1, p.err, 0xB2600003u, abort_flag);
          if (!ok) break;
          load(&tmK, sK + kst * kTile, &k_full[kst], tile_of(j) * BKV, hk, un.b);
          if (j == jb && f.has[u0 ^ 1]) load_q(u0 ^ 1);
          ok = ok && wait_abort(&v_empty[vst], vph ^ 1, p.err, 0xB2600004u, abort_flag);
          if (!ok) break;
          load(&tmV, sV + vst * kTile, &v_full[vst], tile_of(j) * BKV, hk, un.b);
          if (++kst == kK) { kst = 0; kph ^= 1; }
          if (++vst == kV) { vst = 0; vph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------- MMA ----------------------------------
    if (lane == 0) {
      constexpr uint32_t idS = idesc_fmt(BQ, BKV, FMT, false);
      constexpr uint32_t idPV = idesc_fmt(BQ, HD, FMT, true);
      int kst = 0, vst = 0;
      uint32_t kph = 0, vph = 0, qn = 0, pc[2] = {0, 0};
      bool ok = true;
      uint32_t q_at[2] = {0, 0};
      auto issue_s = [&](int u, int j, const Info& g) {
        if (j == g.kb[u]) {  // the unit's first S of this tile: is its Q there?
          q_at[u] = qn % kQ;
          ok = wait_abort(&q_full[q_at[u]], (qn / kQ) & 1, p.err, 0xB2600007u, abort_flag);
          if (!ok) return;
          ++qn;
          tc::fence_after_sync();
        }
#pragma unroll
        for (int kk = 0; kk < HD / Cf::KSTEP; ++kk) {
          const uint64_t da = tc::desc_kmajor_sw128(sQ + q_at[u] * kTile + (kk >> 2) * kAtom + (kk & 3) * 32);
          const uint64_t db = tc::desc_kmajor_sw128(sK + kst * kTile + (kk >> 2) * kAtom + (kk & 3) * 32);
          mma_ss<FMT>(tmem + 256 * u, da, db, idS, kk != 0);
        }
        tc::commit(&s_full[u]);
        if (j == g.nkv[u] - 1) tc::commit(&q_empty[q_at[u]]);
      };
      auto wait_k = [&]() {
        ok = ok && wait_abort(&k_full[kst], kph, p.err, 0xB2600005u, abort_flag);
        if (ok) tc::fence_after_sync();
        return ok;
      };
      auto free_k = [&]() {
        tc::commit(&k_empty[kst]);
        if (++kst == kK) { kst = 0; kph ^= 1; }
      };
      int k = 0;
      auto next_unit = [&](Info& g) {  // the next unit with anything to do
        while (ok && unit_of(p, k, un)) {
          ok = wait_abort(&info_full[k & 1], (k >> 1) & 1, p.err, 0xB2600006u, abort_flag);
          if (!ok) break;
          read_info(k, g);
          mbar_arrive(&info_empty[k & 1]);
          ++k;
          if (g.any()) return true;
        }
        return false;
      };
      // Order: PV_0(j) S_0(j + 1) PV_1(j) S_1(j + 1), where the tile after a
      // unit's last is the next unit's first: one Q tile's softmax warps start on
      // it while the other's are still at the diagonal.  S overwrites P of the
      // tile before, whose PV was issued earlier: MMAs of one thread run in order.
      bool have = next_unit(f);
      if (have && wait_k()) {
        for (int u = 0; u < 2 && ok; ++u)
          if (f.active(u, f.first())) issue_s(u, f.first(), f);
        if (ok) free_k();
      }
      while (ok && have) {
        const int je = f.last();
        Info nx;
        bool more = true;
        for (int j = f.first(); j < je && ok; ++j) {
          int jn = j + 1;
          Info g = f;
          if (jn == je) {
            more = next_unit(nx);
            g = nx;
            jn = more ? nx.first() : 0;
          }
          ok = ok && wait_abort(&v_full[vst], vph, p.err, 0xB2600008u, abort_flag);
          if (!ok) break;
          bool have_k = false;
          for (int u = 0; u < 2 && ok; ++u) {
            if (f.active(u, j)) {
              ok = wait_abort(&p_ready[u], pc[u] & 1, p.err, 0xB2600009u, abort_flag);
              if (!ok) break;
              ++pc[u];
              tc::fence_after_sync();
#pragma unroll
              for (int kk = 0; kk < BKV / Cf::KSTEP; ++kk)
                mma_ts<FMT>(tmem + 256 * u + 128, tmem + 256 * u + p_column(BIAS) + kk * 8,
                            tc::smem_desc(sV + vst * kTile + kk * Cf::KSTEP * 128, kAtom, 1024, tc::kSwizzle128B), idPV,
                            (j != f.kb[u]) || kk != 0);
              if (j == f.nkv[u] - 1) tc::commit(&o_done[u]);
            }
            if (more && g.active(u, jn)) {
              if (!have_k && !wait_k()) break;
              have_k = true;
              issue_s(u, jn, g);
            }
          }
          if (!ok) break;
          tc::commit(&v_empty[vst]);
          if (++vst == kV) { vst = 0; vph ^= 1; }
          if (have_k) free_k();
        }
        f = nx;
        have = more;
      }
      if (!ok) {
        tc::commit(drain);
        mbar_wait(drain, 0, p.err, 0xB260000Au);
      }
    }
  } else if (warp < 4) {
    // ------------------------------- key ranges -------------------------------
    const int t = threadIdx.x - 64;
    auto find = [&](int k) {  // info of turn k
      if (k >= 2 && !__all_sync(0xffffffffu, wait_abort(&info_empty[k & 1], ((k >> 1) - 1) & 1, p.err, 0xB260000Bu, abort_flag)))
        return false;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // smallest / largest first key, largest / smallest end; a row that sees
        // nothing makes every tile a masked one
        int4 x = make_int4(INT_MAX, 0, 0, INT_MAX);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = un.q0 + u * BQ + i * 64 + t;
          if (u < p.per && row < p.Sq) {
            int lo, hi;
            attn::row_range(p.range, un.b, row, p.Skv, lo, hi);
            const bool sees = hi > lo;
            if (sees) x.x = min(x.x, lo);
            x.y = sees ? max(x.y, lo) : INT_MAX;
            if (sees) x.z = max(x.z, hi);
            x.w = sees ? min(x.w, hi) : 0;
          }
        }
        x.x = __reduce_min_sync(0xffffffffu, x.x);
        x.y = __reduce_max_sync(0xffffffffu, x.y);
        x.z = __reduce_max_sync(0xffffffffu, x.z);
        x.w = __reduce_min_sync(0xffffffffu, x.w);
        if (lane == 0) s_info[(k & 1) * 4 + (warp - 2) * 2 + u] = x;
      }
      __syncwarp();
      mbar_arrive(&info_full[k & 1]);
      return true;
    };
    for (int k = 0; unit_of(p, k, un) && find(k); ++k) {
    }
  } else {
    // -------------------------------- softmax --------------------------------
    const int u = (warp - 4) >> 2, qw = warp & 3, r = qw * 32 + lane;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const uint32_t tS = tmem + 256 * u + lane_off, tO = tS + 128;
    Score score = make_score(p.cap);
    uint32_t sc = 0, oc = 0;  // S tiles / outputs waited for
    uint32_t sick = 0;        // turns with a row to look at again (bit 31: all from the 31st on)
    bool ok = true;
    int next_lo = 0, next_hi = 0;
    auto find_row = [&](int k) {  // keys of this thread's row in turn k
      Unit n;
      next_lo = next_hi = 0;
      if (unit_of(p, k, n) && u < p.per && n.q0 + u * BQ + r < p.Sq)
        attn::row_range(p.range, n.b, n.q0 + u * BQ + r, p.Skv, next_lo, next_hi);
    };
    find_row(0);
    for (int k = 0; ok && unit_of(p, k, un); ++k) {
      const int q0 = un.q0 + u * BQ, qpos = q0 + r;
      const bool exists = u < p.per && qpos < p.Sq;
      const int row_lo = next_lo, row_hi = next_hi;
      if constexpr (BIAS) score.slope0 = p.slopes[un.h] * attn::kLog2e;
      ok = __all_sync(0xffffffffu, wait_abort(&info_full[k & 1], (k >> 1) & 1, p.err, 0xB260000Eu, abort_flag));
      if (!ok) break;
      read_info(k, f);
      __syncwarp();
      if (lane == 0) mbar_arrive(&info_empty[k & 1]);
      const int kb = f.kb[u], nkv = f.nkv[u];
      // some tile is masked if the first or the last is
      const bool any_masked = nkv > kb && (f.masked(u, tile_of(kb)) || f.masked(u, tile_of(nkv - 1)));
      float m_used = -INFINITY, l = 0.f;
      for (int j = kb; j < nkv; ++j) {
        ok = __all_sync(0xffffffffu, wait_abort(&s_full[u], sc & 1, p.err, 0xB260000Fu, abort_flag));
        if (!ok) break;
        ++sc;
        tc::fence_after_sync();
        const int kv0 = tile_of(j) * BKV;
        const bool one_side = kv0 + BKV - 1 <= q0 || kv0 >= q0 + BQ - 1;  // where the tile's rows are not in it
        if constexpr (BIAS) {
          score.dist = (float)(qpos - kv0);
          score.slope = kv0 <= q0 ? score.slope0 : -score.slope0;
        }
        uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
        if (f.masked(u, tile_of(j))) range_bits(vis, row_lo, row_hi, kv0);
        const bool whole = (!BIAS || one_side) && whole_tile(vis);
        // O_u is quiescent: PV_u(j-1) finished before S_u(j)
        softmax_tile<true, HD, FMT, CAP, BIAS>(tS, tO, vis, whole, one_side, score, j > kb, m_used, l);
        tmem_st_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[u]);
      }
      if (!ok) break;
      find_row(k + 1);  // under the last PV
      // O_u / l -> global (rows beyond Sq are not stored)
      uint16_t* orow = reinterpret_cast<uint16_t*>(p.o) + un.b * p.os_b + un.h * p.os_h + (int64_t)qpos * p.os_s;
      if (nkv == kb) {  // no row of the tile sees anything: zeros
        if (exists)
          for (int e = 0; e < HD / 8; ++e) reinterpret_cast<uint4*>(orow)[e] = make_uint4(0, 0, 0, 0);
        continue;
      }
      ok = __all_sync(0xffffffffu, wait_abort(&o_done[u], oc & 1, p.err, 0xB2600010u, abort_flag));
      if (!ok) break;
      ++oc;
      tc::fence_after_sync();
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float o[32];
        tc::tmem_ld_32x32b_x32(tO + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(o));
        tc::tmem_ld_wait();
        if ((any_masked || FMT == kF16) && exists) {
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) sum = fmaf(o[e], 0.f, sum);
          // (a row whose weights add up to 0 or NaN is 0 or NaN anyway)
          if (sum != 0.f && l != 0.f && l == l) sick |= 1u << min(k, 31);
        }
        if (l == 0.f) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (exists) {
          uint4* dst = reinterpret_cast<uint4*>(orow + 32 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dst[e] = make_uint4(narrow2<FMT>(o[8 * e] * inv, o[8 * e + 1] * inv),
                                narrow2<FMT>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                narrow2<FMT>(o[8 * e + 4] * inv, o[8 * e + 5] * inv),
                                narrow2<FMT>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
        }
      }
      // the next unit's first PV overwrites O_u once this warpgroup hands over a P
      tc::fence_before_sync();
    }
    // rows looked at again
    if (any_of_softmax(sick != 0) && !any_of_softmax(!ok)) {
      struct Entry {
        int turn, warp;  // u * 4 + qw
        uint32_t rows;
      };
      constexpr int kTurns = (kQ * kTile - 16) / (8 * (int)sizeof(Entry));  // a round's, eight warps each
      int* count = reinterpret_cast<int*>(sQ);
      Entry* list = reinterpret_cast<Entry*>(sQ + 16);
      sick = __reduce_or_sync(0xffffffffu, sick);
      for (int k0 = 0; unit_of(p, k0, un); k0 += kTurns) {
        any_of_softmax(false);  // the round before is over
        if (threadIdx.x == 128) *count = 0;
        any_of_softmax(false);
        for (int k = k0; k < k0 + kTurns && u < p.per && sick >> min(k, 31) && unit_of(p, k, un); ++k) {
          if (!(sick >> min(k, 31) & 1)) continue;
          const uint32_t rows = rows_again<HD, FMT>(p, un, un.q0 + u * BQ, un.q0 + u * BQ + qw * 32);
          if (rows && lane == 0) list[atomicAdd(count, 1)] = {k, u * 4 + qw, rows};
        }
        any_of_softmax(false);
        for (int t = warp - 4, n = 8 * *count; t < n; t += 8) {
          const Entry e = list[t / 8];
          const uint32_t rows = e.rows & 0xfu << t % 8 * 4;
          if (!rows) continue;
          unit_of(p, e.turn, un);
          if constexpr (BIAS) score.slope0 = p.slopes[un.h] * attn::kLog2e;
          compute_rows<HD, FMT, CAP, BIAS>(p, un, un.q0 + e.warp * 32, rows, score);
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

template <int HD, int FMT, bool CAP, bool BIAS>
static void launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const Params& p,
                   cudaStream_t st) {
  constexpr int smem = (kQ + kK + kV) * FaCfg<HD, FMT>::kTile + 1024 + 512;
  const int64_t units = (int64_t)p.n_units * p.Hq * p.B;
  const int grid = (int)(units < num_sms() ? units : num_sms());
  set_max_smem((const void*)scored_kernel<HD, FMT, CAP, BIAS>, smem);
  scored_kernel<HD, FMT, CAP, BIAS><<<grid, kThreads, smem, st>>>(tq, tk, tv, p);
}

}  // namespace scored
}  // namespace b2

using namespace b2;

extern "C" int b2_flash_attn_fwd_scored(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t Hq,
                                        int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D, const int64_t* qs,
                                        const int64_t* ks, const int64_t* vs, const int64_t* os, float scale,
                                        int causal, int64_t window, float softcap, const float* alibi_slopes,
                                        const int32_t* doc_offsets, int64_t n_docs, const int32_t* prefix_lens,
                                        int dtype, void* stream) {
  B2_CHECK_ARG(q && o && qs && ks && vs && os && (Skv == 0 || (k && v)), B2_ERR_INVALID,
               "flash_attn_fwd_scored: null pointer");
  B2_CHECK_ARG(B > 0 && Hq > 0 && Hkv > 0 && Sq >= 0 && Skv >= 0 && D > 0, B2_ERR_INVALID,
               "flash_attn_fwd_scored: bad shape");
  B2_CHECK_ARG(Hq % Hkv == 0, B2_ERR_INVALID, "flash_attn_fwd_scored: Hq=%lld not a multiple of Hkv=%lld",
               (long long)Hq, (long long)Hkv);
  B2_CHECK_ARG((!causal && !doc_offsets) || Sq == Skv, B2_ERR_INVALID,
               "flash_attn_fwd_scored: causal and documents need Sq == Skv");
  B2_CHECK_ARG(window >= 0 && window <= 2147483647 && (!window || causal), B2_ERR_INVALID,
               "flash_attn_fwd_scored: a window needs causal");
  B2_CHECK_ARG(!prefix_lens || (causal && !window), B2_ERR_INVALID,
               "flash_attn_fwd_scored: prefixes need causal and no window");
  B2_CHECK_ARG(!doc_offsets || (n_docs > 0 && n_docs <= 2147483646), B2_ERR_INVALID,
               "flash_attn_fwd_scored: doc_offsets needs n_docs > 0");
  B2_CHECK_ARG(softcap >= 0.f && isfinite(softcap) && isfinite(scale), B2_ERR_INVALID,
               "flash_attn_fwd_scored: scale and softcap must be finite, softcap >= 0");
  B2_CHECK_ARG(dtype == B2_F16 || dtype == B2_BF16 || dtype == B2_F32, B2_ERR_DTYPE, "flash_attn_fwd_scored: dtype %d",
               dtype);
  B2_CHECK_ARG(D <= 256, B2_ERR_UNSUPPORTED, "flash_attn_fwd_scored: D=%lld > 256", (long long)D);
  B2_CHECK_ARG(B <= 65535 && Hq <= 65535 && Sq <= (1 << 24) && Skv <= (1 << 24), B2_ERR_UNSUPPORTED,
               "flash_attn_fwd_scored: sizes too large");
  if (Sq == 0) return B2_OK;
  softcap = attn::cap_in_range(softcap);
  cudaStream_t st = (cudaStream_t)stream;
  attn::RangeMask range;
  range.causal = causal != 0;
  range.window = (int)window;
  range.n_docs = doc_offsets ? (int)n_docs : 0;
  range.docs = doc_offsets;
  range.prefix = prefix_lens;
  bool wide = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(o, 16);
  for (int i = 0; i < 3; ++i) wide = wide && qs[i] % 8 == 0 && ks[i] % 8 == 0 && vs[i] % 8 == 0 && os[i] % 8 == 0;
  // scale > 0: the row maximum is taken before the scale.  fp32 stays fp32 here
  // (the plain kernel reads it as tf32 at head dim 64).  2^20 keys bound the time
  // that rows computed anew may take: 0.3 s for 32 of them over so many.
  unsigned* err = device_error_word();
  if (wide && (D == 64 || D == 128) && dtype != B2_F32 && scale > 0.f && Skv > 0 && err &&
      B * Hq * ((Sq + fa::BQ - 1) / fa::BQ) <= (1 << 30) && Skv <= (1 << 20)) {
    CUtensorMap tq, tk, tv;
    if (make_tmap_4d(&tq, q, dtype, D, Sq, Hq, B, qs) && make_tmap_4d(&tk, k, dtype, D, Skv, Hkv, B, ks) &&
        make_tmap_4d(&tv, v, dtype, D, Skv, Hkv, B, vs)) {
      scored::Params p = {};
      p.B = (int)B;
      p.Hq = (int)Hq;
      p.Hkv = (int)Hkv;
      p.Sq = (int)Sq;
      p.Skv = (int)Skv;
      p.q_tiles = (int)((Sq + fa::BQ - 1) / fa::BQ);
      // Q-tile pairs, or single Q tiles when the pairs would not fill the SMs (causal,
      // cap, 8 heads of 128: 1024 tokens 35 us against 41 in pairs, 2048 55 against 65)
      p.per = (int64_t)((p.q_tiles + 1) / 2) * Hq * B < num_sms() ? 1 : 2;
      p.n_units = (p.q_tiles + p.per - 1) / p.per;
      p.o = o;
      p.os_b = os[0];
      p.os_h = os[1];
      p.os_s = os[2];
      p.err = err;
      p.range = range;
      p.slopes = alibi_slopes;
      p.cap = fa::make_cap(scale, softcap);
      p.q = (const uint16_t*)q;
      p.k = (const uint16_t*)k;
      p.v = (const uint16_t*)v;
      for (int i = 0; i < 3; ++i) {
        p.qs[i] = qs[i];
        p.ks[i] = ks[i];
        p.vs[i] = vs[i];
      }
#define B2_SCORED(HD, FMT)                                                                             \
  do {                                                                                                 \
    if (softcap > 0.f && alibi_slopes) scored::launch<HD, FMT, true, true>(tq, tk, tv, p, st);         \
    else if (softcap > 0.f) scored::launch<HD, FMT, true, false>(tq, tk, tv, p, st);                   \
    else if (alibi_slopes) scored::launch<HD, FMT, false, true>(tq, tk, tv, p, st);                    \
    else scored::launch<HD, FMT, false, false>(tq, tk, tv, p, st);                                     \
  } while (0)
      if (D == 128 && dtype == B2_F16) B2_SCORED(128, fa::kF16);
      else if (D == 128) B2_SCORED(128, fa::kBF16);
      else if (dtype == B2_F16) B2_SCORED(64, fa::kF16);
      else B2_SCORED(64, fa::kBF16);
#undef B2_SCORED
      return launch_status("flash_attn_fwd_scored");
    }
  }
  B2_CHECK_ARG(Sq * (Hq / Hkv) <= 2147483647 - 64, B2_ERR_UNSUPPORTED,
               "flash_attn_fwd_scored: %lld rows a kv head", (long long)(Sq * (Hq / Hkv)));
  attn::SimtParams s = {};
  s.q = q;
  s.k = k;
  s.v = v;
  s.o = o;
  s.B = (int)B;
  s.T = (int)Sq;
  s.Hq = (int)Hq;
  s.Hkv = (int)Hkv;
  s.D = (int)D;
  s.Skv = (int)Skv;
  const int order[3] = {0, 2, 1};  // (b, h, s) -> (b, s, h)
  for (int i = 0; i < 3; ++i) {
    s.qs[i] = qs[order[i]];
    s.os[i] = os[order[i]];
    s.ks[i] = ks[i];
    s.vs[i] = vs[i];
  }
  s.scale = scale;
  s.softcap = softcap;
  s.slopes = alibi_slopes;
  s.range = range;
  s.err = err;
  return attn::launch_simt(s, dtype, dtype, st, "flash_attn_fwd_scored");
}
