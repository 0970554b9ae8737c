// FlashAttention forward with document and prefix masks, capped scores and a
// distance bias: key ranges per row and score forms on the kernels of
// fa_fwd_kernel.cuh (16-bit, head dim 64 / 128, tcgen05) and attn_simt.cu (the
// rest, fp32 arithmetic).  The reference has causal masking only
// (_msl_templates.py:1610-1619).
//
//   s = scale q.k;  softcap: s = softcap tanh(s / softcap);  s -= slope |i - j|
//
// Every mask is one key range per query row (attn::row_range), so a Q tile
// visits the KV tiles from its rows' first visible key to their last and only
// tiles at the ranges' ends are masked.  Capped and biased scores cost softmax
// issue slots, not memory: the cap takes two more MUFU operations a score, the
// bias one more paired FMA.
#include "fa_fwd_kernel.cuh"
#include <math.h>

namespace b2 {

template <int HD, int FMT, bool CAP, bool BIAS>
static void launch_scored(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const fa::Params& p,
                          dim3 grid, cudaStream_t st) {
  using Cf = fa::FaCfg<HD, FMT>;
  set_max_smem((const void*)fa::fa_fwd2_kernel<HD, FMT, true, CAP, BIAS>, (int)Cf::kSmem);
  fa::fa_fwd2_kernel<HD, FMT, true, CAP, BIAS><<<grid, fa::kThreads2, Cf::kSmem, st>>>(tq, tk, tv, p);
}

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
  // (the plain kernel reads it as tf32 at head dim 64).
  unsigned* err = device_error_word();
  if (wide && (D == 64 || D == 128) && dtype != B2_F32 && scale > 0.f && Skv > 0 && err) {
    CUtensorMap tq, tk, tv;
    if (make_tmap_4d(&tq, q, dtype, D, Sq, Hq, B, qs) && make_tmap_4d(&tk, k, dtype, D, Skv, Hkv, B, ks) &&
        make_tmap_4d(&tv, v, dtype, D, Skv, Hkv, B, vs)) {
      fa::Params p = {};
      p.B = (int)B;
      p.Hq = (int)Hq;
      p.Hkv = (int)Hkv;
      p.Sq = (int)Sq;
      p.Skv = (int)Skv;
      p.q_tiles = (int)((Sq + fa::BQ - 1) / fa::BQ);
      p.scale_log2 = scale * fa::kLog2e;
      p.o = o;
      p.os_b = os[0];
      p.os_h = os[1];
      p.os_s = os[2];
      p.err = err;
      p.range = range;
      p.slopes = alibi_slopes;
      p.cap_log2 = softcap * fa::kLog2e;
      p.cap_in = softcap > 0.f ? 2.f * fa::kLog2e * scale / softcap : 0.f;
      p.v = (const uint16_t*)v;
      p.vs_b = vs[0];
      p.vs_h = vs[1];
      p.vs_s = vs[2];
      p.single = (int64_t)((p.q_tiles + 1) / 2) * Hq * B < num_sms() ? 1 : 0;
      const dim3 grid(p.single ? p.q_tiles : (p.q_tiles + 1) / 2, (unsigned)Hq, (unsigned)B);
#define B2_SCORED(HD, FMT)                                                                     \
  do {                                                                                         \
    if (softcap > 0.f && alibi_slopes) launch_scored<HD, FMT, true, true>(tq, tk, tv, p, grid, st);   \
    else if (softcap > 0.f) launch_scored<HD, FMT, true, false>(tq, tk, tv, p, grid, st);      \
    else if (alibi_slopes) launch_scored<HD, FMT, false, true>(tq, tk, tv, p, grid, st);       \
    else launch_scored<HD, FMT, false, false>(tq, tk, tv, p, grid, st);                        \
  } while (0)
      if (D == 128 && dtype == B2_F16) B2_SCORED(128, fa::kF16);
      else if (D == 128) B2_SCORED(128, fa::kBF16);
      else if (dtype == B2_F16) B2_SCORED(64, fa::kF16);
      else B2_SCORED(64, fa::kBF16);
#undef B2_SCORED
      return launch_status("flash_attn_fwd_scored");
    }
  }
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
