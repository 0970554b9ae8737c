// FlashAttention forward (sm_100a): O = softmax(scale * Q K^T [+ causal]) V
//
// Reference: flash_attention template (triton_metal/codegen/_msl_templates.py
// :1568-1767; online softmax m/l/O update at :1697-1753, causal mask
// kv_pos <= q_pos at :1610-1619, final O /= l skipped when l == 0), the
// strided Triton kernel _flash_attn_fwd (tests/test_flash_attention.py:24-104)
// and the GQA head map kv_head = q_head / n_q_per_kv (_msl_templates.py:2101).
//
// Fast path (D = 128, bf16/fp16): one CTA per pair of 128-row Q tiles of one
// (b, h), longest causal pairs first (one Q tile per CTA when the pairs would
// not fill the SMs).
//   warp 0      TMA: both Q tiles once; K tiles (3-stage ring) and V tiles
//               (2-stage) shared by the two Q tiles
//   warp 1      TMEM owner + MMA issuer: S_u = Q_u K^T (M=N=128, K=16 x 8)
//               and O_u += P_u V (P from TMEM, V the MN-major smem B operand)
//               for the two tiles in ping-pong order
//   warps 4-11  two softmax warpgroups (one per Q tile), one query row per
//               thread (TMEM lane = row): row max in the log2 domain,
//               p = exp2(s - m) (a third of them by a polynomial on the
//               FMA pipe, the rest on MUFU), row sum, P as bf16 written back into TMEM
//               over its S columns; O is rescaled in TMEM only when the
//               running max grows by more than 8 (2^8 headroom in P).
//               Final O / l -> global.
// Generic path (any D <= 256, fp32/bf16/fp16, any strides): one warp per
// query row with the same online softmax in fp32.
#include "fa_fwd_kernel.cuh"
#include <string.h>

namespace b2 {
namespace fa {

// ---------------------------------------------------------------------------
// Generic path: one warp per query row, fp32 online softmax (same update as
// the reference template, _msl_templates.py:1712-1743).  Any D <= 256.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float ldf(const T* p) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float*>(p);
  else return to_f32<T>(*p);
}
template <typename T>
__device__ __forceinline__ void stf(T* p, float v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float*>(p) = v;
  else *p = from_f32<T>(v);
}

struct GenParams {
  const void *q, *k, *v;
  void* o;
  int B, Hq, Hkv, Sq, Skv, D, causal;
  int window;  // > 0 (causal only): keys s - window + 1 .. s (sliding window)
  float scale;
  int64_t qs[3], ks[3], vs[3], os[3];
};

template <typename T>
__global__ void __launch_bounds__(128) fa_generic_kernel(const GenParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + warp;
  if (row >= (int64_t)p.B * p.Hq * p.Sq) return;
  const int s = row % p.Sq;
  const int h = (row / p.Sq) % p.Hq;
  const int b = row / ((int64_t)p.Sq * p.Hq);
  const int hk = h / (p.Hq / p.Hkv);
  const T* q = (const T*)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)s * p.qs[2];
  const T* kb = (const T*)p.k + b * p.ks[0] + hk * p.ks[1];
  const T* vb = (const T*)p.v + b * p.vs[0] + hk * p.vs[1];
  constexpr int MAXE = 8;
  float qv[MAXE], acc[MAXE];
#pragma unroll
  for (int e = 0; e < MAXE; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < p.D ? ldf(q + d) * p.scale : 0.f;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int kend = p.causal ? min(p.Skv, s + 1) : p.Skv;
  const int kbeg = p.window > 0 ? max(0, s - p.window + 1) : 0;
  for (int j = kbeg; j < kend; ++j) {
    const T* kr = kb + (int64_t)j * p.ks[2];
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < MAXE; ++e) {
      const int d = lane + 32 * e;
      if (d < p.D) dot += qv[e] * ldf(kr + d);
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float mn = fmaxf(m, dot);
    const float alpha = __expf(m - mn), pj = __expf(dot - mn);
    l = l * alpha + pj;
    const T* vr = vb + (int64_t)j * p.vs[2];
#pragma unroll
    for (int e = 0; e < MAXE; ++e) {
      const int d = lane + 32 * e;
      acc[e] = acc[e] * alpha + (d < p.D ? pj * ldf(vr + d) : 0.f);
    }
    m = mn;
  }
  T* o = (T*)p.o + b * p.os[0] + h * p.os[1] + (int64_t)s * p.os[2];
  const float inv = l > 0.f ? 1.f / l : 0.f;  // all-masked row -> 0 (reference nan_to_num)
#pragma unroll
  for (int e = 0; e < MAXE; ++e) {
    const int d = lane + 32 * e;
    if (d < p.D) stf(o + d, acc[e] * inv);
  }
}

}  // namespace fa

template <int HD, int FMT>
static void launch_fa_tc(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const fa::Params& p,
                         dim3 grid, cudaStream_t st) {
  using Cf = fa::FaCfg<HD, FMT>;
  set_max_smem((const void*)fa::fa_fwd2_kernel<HD, FMT, false, false, false>, (int)Cf::kSmem);
  fa::fa_fwd2_kernel<HD, FMT, false, false, false><<<grid, fa::kThreads2, Cf::kSmem, st>>>(tq, tk, tv, p);
}

}  // namespace b2

using namespace b2;

static int launch_fa_generic(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t Hq,
                             int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D, const int64_t* qs, const int64_t* ks,
                             const int64_t* vs, const int64_t* os, float scale, int causal, int window, int dtype,
                             cudaStream_t st) {
  fa::GenParams g;
  g.q = q;
  g.k = k;
  g.v = v;
  g.o = o;
  g.B = (int)B;
  g.Hq = (int)Hq;
  g.Hkv = (int)Hkv;
  g.Sq = (int)Sq;
  g.Skv = (int)Skv;
  g.D = (int)D;
  g.causal = causal;
  g.window = window;
  g.scale = scale;
  for (int i = 0; i < 3; ++i) {
    g.qs[i] = qs[i];
    g.ks[i] = ks[i];
    g.vs[i] = vs[i];
    g.os[i] = os[i];
  }
  const int64_t rows = B * Hq * Sq;
  const unsigned blocks = (unsigned)((rows + 3) / 4);
  if (dtype == B2_F32) fa::fa_generic_kernel<float><<<blocks, 128, 0, st>>>(g);
  else if (dtype == B2_BF16) fa::fa_generic_kernel<__nv_bfloat16><<<blocks, 128, 0, st>>>(g);
  else fa::fa_generic_kernel<__half><<<blocks, 128, 0, st>>>(g);
  return launch_status("fa_generic");
}

static int fa_fwd_impl(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t Hq, int64_t Hkv,
                       int64_t Sq, int64_t Skv, int64_t D, const int64_t* qs, const int64_t* ks, const int64_t* vs,
                       const int64_t* os, float scale, int causal, int window, int dtype, void* stream) {
  B2_CHECK_ARG(q && k && v && o && qs && ks && vs && os, B2_ERR_INVALID, "flash_attn_fwd: null pointer");
  B2_CHECK_ARG(B > 0 && Hq > 0 && Hkv > 0 && Sq >= 0 && Skv >= 0 && D > 0, B2_ERR_INVALID,
               "flash_attn_fwd: bad shape");
  B2_CHECK_ARG(Hq % Hkv == 0, B2_ERR_INVALID, "flash_attn_fwd: Hq=%lld not a multiple of Hkv=%lld", (long long)Hq,
               (long long)Hkv);
  B2_CHECK_ARG(!causal || Sq == Skv, B2_ERR_INVALID, "flash_attn_fwd: causal needs Sq == Skv (square tril mask)");
  B2_CHECK_ARG(dtype == B2_F16 || dtype == B2_BF16 || dtype == B2_F32, B2_ERR_DTYPE, "flash_attn_fwd: dtype %d",
               dtype);
  B2_CHECK_ARG(D <= 256, B2_ERR_UNSUPPORTED, "flash_attn_fwd: D=%lld > 256", (long long)D);
  if (Sq == 0) return B2_OK;
  cudaStream_t st = (cudaStream_t)stream;
  // tcgen05 path: D = 128 with 16-bit operands, D = 64 with 16-bit operands or
  // fp32 (read as tf32, fp32 output); TMA-able strides and base addresses
  const bool shape_ok = (D == 128 && dtype != B2_F32) || D == 64;
  const bool fast = shape_ok && Skv > 0 && strides_ok(qs, dtype) && strides_ok(ks, dtype) && strides_ok(vs, dtype) &&
                    strides_ok(os, dtype) && aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(o, 16) &&
                    B <= 65535 && Hq <= 65535;
  if (fast) {
    unsigned* err = device_error_word();
    CUtensorMap tq, tk, tv;
    if (err && make_tmap_4d(&tq, q, dtype, D, Sq, Hq, B, qs) && make_tmap_4d(&tk, k, dtype, D, Skv, Hkv, B, ks) &&
        make_tmap_4d(&tv, v, dtype, D, Skv, Hkv, B, vs, dtype == B2_F32)) {
      fa::Params p = {};
      p.B = (int)B;
      p.Hq = (int)Hq;
      p.Hkv = (int)Hkv;
      p.Sq = (int)Sq;
      p.Skv = (int)Skv;
      p.causal = causal;
      p.window = window;
      p.q_tiles = (int)((Sq + fa::BQ - 1) / fa::BQ);
      p.scale_log2 = scale * fa::kLog2e;
      p.o = o;
      p.os_b = os[0];
      p.os_h = os[1];
      p.os_s = os[2];
      p.err = err;
      // Q-tile pairs, or single Q tiles when the pairs would not fill the SMs
      p.single = (int64_t)((p.q_tiles + 1) / 2) * Hq * B < num_sms() ? 1 : 0;
      dim3 grid(p.single ? p.q_tiles : (p.q_tiles + 1) / 2, (unsigned)Hq, (unsigned)B);
      if (D == 128) {
        if (dtype == B2_F16) launch_fa_tc<128, fa::kF16>(tq, tk, tv, p, grid, st);
        else launch_fa_tc<128, fa::kBF16>(tq, tk, tv, p, grid, st);
      } else {
        if (dtype == B2_F16) launch_fa_tc<64, fa::kF16>(tq, tk, tv, p, grid, st);
        else if (dtype == B2_BF16) launch_fa_tc<64, fa::kBF16>(tq, tk, tv, p, grid, st);
        else launch_fa_tc<64, fa::kTF32>(tq, tk, tv, p, grid, st);
      }
      return launch_status("fa_fwd");
    }
  }
  return launch_fa_generic(q, k, v, o, B, Hq, Hkv, Sq, Skv, D, qs, ks, vs, os, scale, causal, window, dtype, st);
}

extern "C" int b2_flash_attn_fwd(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t Hq,
                                 int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D, const int64_t* qs,
                                 const int64_t* ks, const int64_t* vs, const int64_t* os, float scale, int causal,
                                 int dtype, void* stream) {
  return fa_fwd_impl(q, k, v, o, B, Hq, Hkv, Sq, Skv, D, qs, ks, vs, os, scale, causal, 0, dtype, stream);
}

// Causal sliding-window FlashAttention (Mistral-style): query s attends to
// keys s - window + 1 .. s.  The prefill counterpart of the decode window
// (sliding_window_attention, _msl_templates.py:3335-3431).  Same dispatch as
// b2_flash_attn_fwd: the tcgen05 kernel for D = 128 bf16/fp16 (each Q tile
// visits only the KV tiles its window reaches), else the CUDA-core kernel.
extern "C" int b2_flash_attn_fwd_window(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t Hq,
                                        int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D, const int64_t* qs,
                                        const int64_t* ks, const int64_t* vs, const int64_t* os, float scale,
                                        int64_t window, int dtype, void* stream) {
  B2_CHECK_ARG(window > 0 && window <= 2147483647, B2_ERR_INVALID, "flash_attn_fwd_window: window must be > 0");
  return fa_fwd_impl(q, k, v, o, B, Hq, Hkv, Sq, Skv, D, qs, ks, vs, os, scale, 1, (int)window, dtype, stream);
}
