// Attention on the CUDA cores with fp32 arithmetic: any head dim up to 256,
// any of the three types (queries and cache may differ), contiguous or paged
// K/V, drafted-token trees or key ranges per row, capped and biased scores.
// It serves what the tensor-core kernels do not take: fp32 (kept in fp32, not
// rounded to tf32), odd head dims, mixed types, unaligned rows.
//
//   s = scale q.k;  s = cap tanh(s / cap);  s -= slope |i - j|
//   o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m}   over the visible keys
//
// A CTA takes 32 rows (query position x query head of one kv head, so that a
// K/V row read once serves all of them) and walks its keys in tiles of 64 kept
// in shared memory as fp32.  Each thread makes a 4 x 4 block of scores and a
// 4 x (D / 16) block of outputs in registers: 8 16-byte shared loads for 64
// FMAs in either product, so the FMA pipe sets the pace, not shared memory.
// Few rows and long caches: the keys are split over CTAs and the partials
// (m, l, unnormalised o) are joined by a second kernel.  Trees of 5 over three
// requests of up to 777 keys, 8 heads of 64, fp32, capped: 25 us a call (38 with
// 4-byte loads), the latency of a CTA's few tiles and of the join.
#include "attn_common.cuh"

namespace b2 {
namespace attn {

constexpr int kThreads = 128;
constexpr int BM = 32, BN = 64;

template <typename T>
__device__ __forceinline__ float ldf(const T* p) {
  return to_f32<T>(*p);
}

template <int DP>
struct SimtCfg {
  static constexpr int LD = DP + 4;  // rows 16-byte aligned, 8 neighbours in different banks
  static constexpr int kSmem = (BM * DP + 2 * BN * LD + BM * (BN + 4)) * 4 + BM * 8 + BN * 16;
};

template <typename TQ, typename TKV, int DP>
__global__ void __launch_bounds__(kThreads) simt_kernel(const SimtParams p) {
  using C = SimtCfg<DP>;
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;                  // [BM][DP], scaled
  float* sK = sQ + BM * DP;        // [BN][LD]
  float* sV = sK + BN * C::LD;     // [BN][LD]
  float* sP = sV + BN * C::LD;     // [BM][BN + 4]
  int* sLo = reinterpret_cast<int*>(sP + BM * (BN + 4));  // key range of each row (tree: of the context)
  int* sHi = sLo + BM;
  int64_t* sOff = reinterpret_cast<int64_t*>(sHi + BM);   // K / V row offsets of the tile's keys, -1: zeros
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int rep = p.Hq / p.Hkv, R = p.T * rep;
  const int split = blockIdx.x % p.nsplit, r0 = blockIdx.x / p.nsplit * BM;
  const int hk = blockIdx.y, b = blockIdx.z;
  const bool tree = p.tree_mask != nullptr;
  int ctx = 0, dl = 0;
  if (tree) tree_lens(p.ctx, p.draft, b, p.T, p.Skv, ctx, dl);

  if (tid < BM) {
    const int r = r0 + tid;
    int lo = 0, hi = 0;
    if (r < R) {
      if (!tree) row_range(p.range, b, r / rep, p.Skv, lo, hi);
      else if (r / rep < dl) hi = ctx + dl;
    }
    sLo[tid] = lo;
    sHi[tid] = hi;
  }
  for (int e = tid; e < BM * DP; e += kThreads) {
    const int r = r0 + e / DP, d = e % DP;
    float val = 0.f;
    if (r < R && d < p.D)
      val = ldf((const TQ*)p.q + b * p.qs[0] + (int64_t)(r / rep) * p.qs[1] + (int64_t)(hk * rep + r % rep) * p.qs[2] + d);
    sQ[e] = val * p.scale;
  }
  __syncthreads();
  // keys that some row of the tile sees, and this split's share of them
  int k_lo = 0x7fffffff, k_hi = 0;
  for (int i = 0; i < BM; ++i)
    if (sHi[i] > sLo[i]) {
      k_lo = min(k_lo, sLo[i]);
      k_hi = max(k_hi, sHi[i]);
    }
  if (k_hi == 0) k_lo = 0;
  int s0 = k_lo, s1 = k_hi;
  if (p.nsplit > 1) {
    s0 = min(k_hi, k_lo + split * p.split_len);
    s1 = min(k_hi, s0 + p.split_len);
  }

  float m[4], l[4], acc[4][DP / 16];
  int row_q[4];  // query position, for the distance bias and the tree mask
  float slope[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    const int r = min(r0 + ty * 4 + i, R - 1);
    row_q[i] = r / rep;
    slope[i] = p.slopes ? p.slopes[hk * rep + r % rep] : 0.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) acc[i][d] = 0.f;
  }
  const uint8_t* tmask = tree ? p.tree_mask + b * p.tree_stride : nullptr;

  for (int t0 = s0; t0 < s1; t0 += BN) {
    __syncthreads();  // the previous tile is consumed
    if (tid < BN) {
      const int pos = t0 + tid;
      int64_t ko = -1, vo = -1;
      if (pos < s1) {
        if (p.page_table) {
          const int pg = p.page_table[(int64_t)b * p.max_pages + pos / p.page_size];
          const int off = pos % p.page_size;
          if (pg >= 0 && pg < p.n_pages) {
            ko = pg * p.ks[0] + off * p.ks[1] + hk * p.ks[2];
            vo = pg * p.vs[0] + off * p.vs[1] + hk * p.vs[2];
          } else {
            atomicCAS(p.err, 0u, kErrPage);  // the key reads as zeros
          }
        } else {
          ko = b * p.ks[0] + hk * p.ks[1] + (int64_t)pos * p.ks[2];
          vo = b * p.vs[0] + hk * p.vs[1] + (int64_t)pos * p.vs[2];
        }
      }
      sOff[tid] = ko;
      sOff[BN + tid] = vo;
    }
    __syncthreads();
    int odd = 0;  // a V value that is not finite
    // the tile: 16-byte loads, eight of K and of V in flight a thread, where rows
    // start on 16 bytes and are whole vectors long, else one value at a time
    constexpr int VE = 16 / (int)sizeof(TKV), VR = DP / VE;  // values of a vector, vectors of a row
    if (p.wide) {
#pragma unroll 1
      for (int e0 = tid; e0 < BN * VR; e0 += 8 * kThreads) {
        uint4 a[8], c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int e = e0 + u * kThreads, j = e / VR, d = e % VR * VE;
          const bool there = e < BN * VR && d < p.D && sOff[j] >= 0;
          a[u] = there ? *reinterpret_cast<const uint4*>((const TKV*)p.k + sOff[j] + d) : make_uint4(0, 0, 0, 0);
          c[u] = there ? *reinterpret_cast<const uint4*>((const TKV*)p.v + sOff[BN + j] + d) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int e = e0 + u * kThreads, j = e / VR, d = e % VR * VE;
          if (e >= BN * VR) break;
          const TKV* ka = reinterpret_cast<const TKV*>(&a[u]);
          const TKV* va = reinterpret_cast<const TKV*>(&c[u]);
#pragma unroll
          for (int x = 0; x < VE; x += 4) {
            const float4 kf = make_float4(ldf(ka + x), ldf(ka + x + 1), ldf(ka + x + 2), ldf(ka + x + 3));
            const float4 vf = make_float4(ldf(va + x), ldf(va + x + 1), ldf(va + x + 2), ldf(va + x + 3));
            odd |= !(fabsf(vf.x) < INFINITY) | !(fabsf(vf.y) < INFINITY) | !(fabsf(vf.z) < INFINITY) | !(fabsf(vf.w) < INFINITY);
            *reinterpret_cast<float4*>(sK + j * C::LD + d + x) = kf;
            *reinterpret_cast<float4*>(sV + j * C::LD + d + x) = vf;
          }
        }
      }
    }
    for (int e = tid; e < (p.wide ? 0 : BN * DP); e += kThreads) {
      const int j = e / DP, d = e % DP;
      float kv = 0.f, vv = 0.f;
      if (d < p.D && sOff[j] >= 0) {
        kv = ldf((const TKV*)p.k + sOff[j] + d);
        vv = ldf((const TKV*)p.v + sOff[BN + j] + d);
      }
      odd |= !(fabsf(vv) < INFINITY);
      sK[j * C::LD + d] = kv;
      sV[j * C::LD + d] = vv;
    }
    odd = __syncthreads_or(odd);
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    for (int d = 0; d < DP; d += 4) {
      float4 a[4], c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sQ + (ty * 4 + i) * DP + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * C::LD + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(a[i].x, c[j].x, s[i][j]);
          s[i][j] = fmaf(a[i].y, c[j].y, s[i][j]);
          s[i][j] = fmaf(a[i].z, c[j].z, s[i][j]);
          s[i][j] = fmaf(a[i].w, c[j].w, s[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = ty * 4 + i, lo = sLo[rr], hi = sHi[rr];
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = t0 + tx + 16 * j;
        float x = s[i][j];
        if (p.softcap > 0.f) x = p.softcap * tanh_acc(__fdividef(x, p.softcap));
        if (p.slopes) x = fmaf(-slope[i], fabsf((float)(row_q[i] - key)), x);
        bool vis = key >= lo && key < hi && key < s1;
        if (tree && vis && key >= ctx) vis = tmask[(int64_t)row_q[i] * p.T + key - ctx] != 0;
        s[i][j] = vis ? x : -INFINITY;
        mx = fmaxf(mx, s[i][j]);  // drops a NaN; its weight is NaN below, as the formula's
      }
#pragma unroll
      for (int off = 8; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float mn = fmaxf(m[i], mx), ref = mn == -INFINITY ? 0.f : mn;
      const float rl = ref * kLog2e;
      // exponent: fma of the score, so that only the small difference rounds
      const float alpha = m[i] == -INFINITY ? 0.f : exp2f(fmaf(m[i], kLog2e, -rl));
      float ts = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // -0: a key that the row does not see
        const float e = s[i][j] == -INFINITY ? -0.f : exp2f(fmaf(s[i][j], kLog2e, -rl));
        ts += e;
        sP[rr * (BN + 4) + tx + 16 * j] = e;
      }
#pragma unroll
      for (int off = 8; off; off >>= 1) ts += __shfl_xor_sync(0xffffffffu, ts, off);
      l[i] = fmaf(l[i], alpha, ts);
      m[i] = mn;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) acc[i][d] *= alpha;
    }
    __syncwarp();  // a warp's 8 rows of P are its own
    if (!odd) {
      for (int j = 0; j < BN; j += 4) {
        float4 pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = *reinterpret_cast<const float4*>(sP + (ty * 4 + i) * (BN + 4) + j);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
          for (int dd = 0; dd < DP / 64; ++dd) {
            const float4 vv = *reinterpret_cast<const float4*>(sV + (j + jj) * C::LD + 64 * dd + 4 * tx);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float pj = jj == 0 ? pr[i].x : jj == 1 ? pr[i].y : jj == 2 ? pr[i].z : pr[i].w;
              acc[i][4 * dd] = fmaf(pj, vv.x, acc[i][4 * dd]);
              acc[i][4 * dd + 1] = fmaf(pj, vv.y, acc[i][4 * dd + 1]);
              acc[i][4 * dd + 2] = fmaf(pj, vv.z, acc[i][4 * dd + 2]);
              acc[i][4 * dd + 3] = fmaf(pj, vv.w, acc[i][4 * dd + 3]);
            }
          }
      }
    } else {
      // some V of the tile is infinite or NaN: one that the row does not see must be
      // dropped, not multiplied by 0, and one that it sees counts whatever its weight
      // (0 where the score is too far below the largest)
      for (int j = 0; j < BN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pj = sP[(ty * 4 + i) * (BN + 4) + j];
          if (__float_as_uint(pj) != 0x80000000u)
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
              const float vv = sV[j * C::LD + 64 * (d >> 2) + 4 * tx + (d & 3)];
              if (pj != 0.f) acc[i][d] = fmaf(pj, vv, acc[i][d]);
              else if (!(fabsf(vv) < INFINITY)) acc[i][d] += vv;
            }
        }
    }
  }

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + ty * 4 + i;
    if (r >= R) continue;
    const int s = r / rep, hq = hk * rep + r % rep;
    if (p.nsplit == 1) {
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      TQ* o = (TQ*)p.o + b * p.os[0] + s * p.os[1] + hq * p.os[2];
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const int dd = 64 * (d >> 2) + 4 * tx + (d & 3);
        if (dd < p.D) o[dd] = from_f32<TQ>(acc[i][d] * inv);
      }
    } else {
      float* w = p.ws + (((((int64_t)b * p.Hkv + hk) * R) + r) * p.nsplit + split) * (p.D + 2);
      if (tx == 0) {
        w[0] = m[i];
        w[1] = l[i];
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const int dd = 64 * (d >> 2) + 4 * tx + (d & 3);
        if (dd < p.D) w[2 + dd] = acc[i][d];
      }
    }
  }
}

// o = sum_s e^{m_s - M} o_s / sum_s e^{m_s - M} l_s over the splits of one row
template <typename TQ>
__global__ void simt_combine_kernel(const SimtParams p) {
  const int rep = p.Hq / p.Hkv;
  const int64_t R = (int64_t)p.T * rep, row = blockIdx.x;
  const int r = (int)(row % R), hk = (int)(row / R % p.Hkv), b = (int)(row / R / p.Hkv);
  const float* w = p.ws + row * p.nsplit * (p.D + 2);
  float M = -INFINITY;
  for (int s = 0; s < p.nsplit; ++s) M = fmaxf(M, w[s * (p.D + 2)]);
  TQ* o = (TQ*)p.o + b * p.os[0] + (r / rep) * p.os[1] + (int64_t)(hk * rep + r % rep) * p.os[2];
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float num = 0.f, den = 0.f;
    for (int s = 0; s < p.nsplit; ++s) {
      const float* ws = w + s * (p.D + 2);
      if (ws[1] == 0.f) continue;  // saw nothing
      const float f = exp2f((ws[0] - M) * kLog2e);
      num = fmaf(f, ws[2 + d], num);
      den = fmaf(f, ws[1], den);
    }
    o[d] = from_f32<TQ>(den == 0.f ? 0.f : num / den);
  }
}

// Splits: about 2 CTAs an SM, each with at least two tiles of keys.
int simt_splits(int64_t row_tiles, int64_t max_keys) {
  const int64_t want = 2 * num_sms();
  if (row_tiles >= want) return 1;
  int64_t ns = (want + row_tiles - 1) / row_tiles;
  const int64_t most = (max_keys + 2 * BN - 1) / (2 * BN);
  if (ns > most) ns = most;
  return ns < 1 ? 1 : (int)ns;
}

size_t simt_workspace(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_keys) {
  const int64_t tiles = B * Hkv * ((T * (Hq / Hkv) + BM - 1) / BM);
  const int ns = simt_splits(tiles, max_keys);
  return ns == 1 ? 0 : (size_t)B * Hq * T * ns * (D + 2) * sizeof(float);
}

template <typename TQ, typename TKV>
static void launch_dp(const SimtParams& p, dim3 grid, cudaStream_t st) {
#define B2_SIMT(DP)                                                                        \
  do {                                                                                     \
    set_max_smem((const void*)simt_kernel<TQ, TKV, DP>, SimtCfg<DP>::kSmem);               \
    simt_kernel<TQ, TKV, DP><<<grid, kThreads, SimtCfg<DP>::kSmem, st>>>(p);               \
  } while (0)
  if (p.D <= 64) B2_SIMT(64);
  else if (p.D <= 128) B2_SIMT(128);
  else B2_SIMT(256);
#undef B2_SIMT
}

// Checked sizes come in; p.ws holds simt_workspace(...) bytes when that is not 0
// (null: one split).
int launch_simt(SimtParams p, int q_dtype, int kv_dtype, cudaStream_t st, const char* what) {
  const int64_t rows = (int64_t)p.T * (p.Hq / p.Hkv), tiles = (rows + BM - 1) / BM;
  p.nsplit = p.ws ? simt_splits(tiles * p.B * p.Hkv, p.Skv) : 1;
  p.split_len = (int)(((int64_t)p.Skv + p.nsplit - 1) / p.nsplit);
  p.split_len = (p.split_len + BN - 1) / BN * BN;
  const int es = kv_dtype == B2_F32 ? 4 : 2;
  p.wide = p.D * es % 16 == 0 && aligned(p.k, 16) && aligned(p.v, 16);
  for (int i = 0; i < 3; ++i) p.wide = p.wide && p.ks[i] * es % 16 == 0 && p.vs[i] * es % 16 == 0;
  const dim3 grid((unsigned)(tiles * p.nsplit), p.Hkv, p.B);
#define B2_SIMT_KV(TQ)                                             \
  do {                                                             \
    if (kv_dtype == B2_F32) launch_dp<TQ, float>(p, grid, st);     \
    else if (kv_dtype == B2_F16) launch_dp<TQ, __half>(p, grid, st); \
    else launch_dp<TQ, __nv_bfloat16>(p, grid, st);                \
    if (p.nsplit > 1)                                              \
      simt_combine_kernel<TQ><<<(unsigned)(rows * p.Hkv * p.B), 128, 0, st>>>(p); \
  } while (0)
  if (q_dtype == B2_F32) B2_SIMT_KV(float);
  else if (q_dtype == B2_F16) B2_SIMT_KV(__half);
  else B2_SIMT_KV(__nv_bfloat16);
#undef B2_SIMT_KV
  return launch_status(what);
}

}  // namespace attn
}  // namespace b2
