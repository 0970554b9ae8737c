// Attention of a tree of drafted tokens over a contiguous or paged KV cache.
#include "attn_common.cuh"
#include <math.h>

using namespace b2;

extern "C" size_t b2_tree_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                              int64_t max_keys, int q_dtype, int kv_dtype) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_keys <= 0) return 0;
  return attn::simt_workspace(B, T, Hq, Hkv, D, max_keys);
}

extern "C" int b2_tree_attn(const void* q, const void* k, const void* v, void* o, const int32_t* page_table,
                            const int32_t* context_lens, const int32_t* draft_lens, const uint8_t* tree_mask,
                            int64_t mask_stride, void* workspace, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                            int64_t D, int64_t max_keys, int64_t page_size, int64_t max_pages, int64_t n_pages,
                            const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                            const int64_t* o_strides, float scale, float softcap, int q_dtype, int kv_dtype,
                            void* stream) {
  B2_CHECK_ARG(B >= 0 && T >= 0 && Hq > 0 && Hkv > 0 && D > 0 && max_keys >= 0, B2_ERR_INVALID,
               "tree_attn: bad shape");
  B2_CHECK_ARG(Hq % Hkv == 0, B2_ERR_INVALID, "tree_attn: Hq=%lld not a multiple of Hkv=%lld", (long long)Hq,
               (long long)Hkv);
  B2_CHECK_ARG(D <= 256, B2_ERR_UNSUPPORTED, "tree_attn: D=%lld > 256", (long long)D);
  B2_CHECK_ARG(B <= 65535 && Hkv <= 65535 && T * (Hq / Hkv) <= (1 << 24) && max_keys <= 2000000000 &&
                   B * Hq * T <= 2147483647,
               B2_ERR_UNSUPPORTED, "tree_attn: sizes too large");
  B2_CHECK_ARG((q_dtype == B2_F32 || q_dtype == B2_F16 || q_dtype == B2_BF16) &&
                   (kv_dtype == B2_F32 || kv_dtype == B2_F16 || kv_dtype == B2_BF16),
               B2_ERR_DTYPE, "tree_attn: dtypes %d / %d", q_dtype, kv_dtype);
  B2_CHECK_ARG(softcap >= 0.f && isfinite(softcap) && isfinite(scale), B2_ERR_INVALID,
               "tree_attn: scale and softcap must be finite, softcap >= 0");
  B2_CHECK_ARG(mask_stride == 0 || mask_stride == T * T, B2_ERR_INVALID, "tree_attn: mask_stride must be 0 or T * T");
  if (B == 0 || T == 0) return B2_OK;
  B2_CHECK_ARG(q && o && context_lens && tree_mask && q_strides && k_strides && v_strides && o_strides &&
                   (max_keys == 0 || (k && v)),
               B2_ERR_INVALID, "tree_attn: null pointer");
  B2_CHECK_ARG(page_size == 0 || (page_size > 0 && page_table && max_pages > 0 && n_pages >= 0 &&
                                  max_keys <= page_size * max_pages),
               B2_ERR_INVALID, "tree_attn: a paged cache needs page_table and max_keys <= max_pages * page_size");
  attn::SimtParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = o;
  p.B = (int)B;
  p.T = (int)T;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.D = (int)D;
  p.Skv = (int)max_keys;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = o_strides[i];
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  p.page_table = page_size ? page_table : nullptr;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages;
  p.n_pages = n_pages;
  p.scale = scale;
  p.softcap = softcap;
  p.tree_mask = tree_mask;
  p.tree_stride = mask_stride;
  p.ctx = context_lens;
  p.draft = draft_lens;
  p.err = device_error_word();
  B2_CHECK_ARG(p.err, B2_ERR_LAUNCH, "tree_attn: no device");
  const size_t need = b2_tree_attn_workspace_size(B, T, Hq, Hkv, D, max_keys, q_dtype, kv_dtype);
  B2_CHECK_ARG(need == 0 || workspace, B2_ERR_INVALID, "tree_attn: workspace required");
  p.ws = need ? (float*)workspace : nullptr;
  return attn::launch_simt(p, q_dtype, kv_dtype, (cudaStream_t)stream, "tree_attn");
}
