// Attention of a tree of drafted tokens over a contiguous or paged KV cache:
// entry points and the TMA form (tree_attn_kernel.cuh has the kernel).
#include "tree_attn_kernel.cuh"

namespace b2 {
namespace tree {

static bool make_map(CUtensorMap* map, const void* base, bool f16, const uint64_t (&dims)[4],
                     const int64_t (&strides)[3], uint32_t box1, uint32_t box2) {
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (EncodeFn) nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  if (!fn) return false;
  const cuuint64_t d[4] = {dims[0], dims[1], dims[2], dims[3]};
  const cuuint64_t st[3] = {(cuuint64_t)strides[0] * 2, (cuuint64_t)strides[1] * 2, (cuuint64_t)strides[2] * 2};
  const cuuint32_t box[4] = {64, box1, box2, 1}, one[4] = {1, 1, 1, 1};
  return fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base),
            d, st, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_maps(Maps& m, const Params& p, int64_t D, int64_t Hq, bool f16) {
  const uint64_t d = (uint64_t)D;
  if (!make_map(&m.q, p.q, f16, {d, (uint64_t)Hq, (uint64_t)p.T, (uint64_t)p.B}, {p.qs[2], p.qs[1], p.qs[0]}, p.rep,
                p.tpt))
    return false;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? p.vs : p.ks;
    CUtensorMap* map = i ? &m.v : &m.k;
    const void* base = i ? p.v : p.k;
    const bool ok = p.page_size
                        ? make_map(map, base, f16, {d, (uint64_t)p.Hkv, p.page_size, (uint64_t)p.n_pages}, {s[2], s[1], s[0]}, 1,
                                   p.box)
                        : make_map(map, base, f16, {d, (uint64_t)p.cap, (uint64_t)p.Hkv, (uint64_t)p.B}, {s[2], s[1], s[0]},
                                   p.box, 1);
    if (!ok) return false;
  }
  return true;
}

int box_of(int64_t page_size, int64_t n_pages) {
  if (!page_size) return BK;
  if (n_pages <= 0) return 0;
  int box = BK;
  while (box && page_size % box) box /= 2;
  return box >= 8 ? box : 0;  // a swizzle atom has 8 rows
}

void launch_any(const Params& p, int64_t D, int64_t Hq, bool f16, bool pair, cudaStream_t st) {
  Maps m = {};
  if (!p.box || !make_maps(m, p, D, Hq, f16)) launch_cp(m, p, (int)D, f16, pair, st);
  else launch_tma(m, p, (int)D, f16, pair, st);
}

void launch_tma(const Maps& m, const Params& p, int D, bool f16, bool pair, cudaStream_t st) {
  launch_form<true>(m, p, D, f16, pair, st);
}

size_t workspace(int64_t T, int64_t rep, int64_t D) {
  const int64_t rows = rep > BR || T > BR / rep ? 2 * BR : BR;
  return (size_t)2 * num_sms() * rows * (D + 2) * sizeof(float);
}

}  // namespace tree
}  // namespace b2

using namespace b2;

// The tensor-core kernel takes 16-bit queries and cache of one type with head
// dim 64 or 128; the rest runs on the CUDA cores.
static bool tree_tc(int64_t D, int q_dtype, int kv_dtype) {
  return q_dtype == kv_dtype && q_dtype != B2_F32 && (D == 64 || D == 128);
}

extern "C" size_t b2_tree_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                              int64_t max_keys, int q_dtype, int kv_dtype) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_keys <= 0) return 0;
  const size_t simt = attn::simt_workspace(B, T, Hq, Hkv, D, max_keys);
  if (!tree_tc(D, q_dtype, kv_dtype)) return simt;
  // the larger of both kernels' needs, since strides and alignment, which also
  // decide, come with the call
  const size_t tc = tree::workspace(T, Hq / Hkv, D);
  return tc > simt ? tc : simt;
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
  softcap = attn::cap_in_range(softcap);
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
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t rep = Hq / Hkv;
  bool wide = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(o, 16) && aligned(workspace, 16);
  for (int i = 0; i < 3; ++i)
    wide = wide && q_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0 && o_strides[i] % 8 == 0;
  const int copies = tree::copies_of(T * rep);
  const int64_t tpt = rep <= tree::BR ? tree::BR / copies / rep : 0;
  const bool pair = T > tpt;
  const int64_t n_rt = tpt ? (T + tpt * (pair ? 2 : 1) - 1) / (tpt * (pair ? 2 : 1)) : 0;
  // scale > 0: the row maximum is taken before the scale
  if (tree_tc(D, q_dtype, kv_dtype) && wide && tpt && scale > 0.f && max_keys > 0 &&
      Hkv * n_rt * ((max_keys + tree::BK - 1) / tree::BK + tree::kItemCost) <= (1 << 30) && n_rt * Hkv <= (1 << 24)) {
    tree::Params t = {};
    t.q = (const uint16_t*)q;
    t.k = (const uint16_t*)k;
    t.v = (const uint16_t*)v;
    t.o = (uint16_t*)o;
    t.page_table = page_table;
    t.ctx = context_lens;
    t.draft = draft_lens;
    t.mask = tree_mask;
    t.ws = (float*)workspace;
    t.mask_stride = mask_stride;
    t.n_pages = page_size ? n_pages : B;
    for (int i = 0; i < 3; ++i) {
      t.qs[i] = q_strides[i];
      t.os[i] = o_strides[i];
      t.ks[i] = k_strides[i];
      t.vs[i] = v_strides[i];
    }
    t.B = (int)B;
    t.T = (int)T;
    t.Hkv = (int)Hkv;
    t.rep = (int)rep;
    t.cap = (int)max_keys;
    t.tpt = (int)tpt;
    t.copies = copies;
    t.n_rt = (int)n_rt;
    t.page_size = (uint32_t)page_size;
    t.max_pages = (int)max_pages;
    t.softcap = fa::make_cap(scale, softcap);
    t.err = p.err;
    t.box = tree::box_of(page_size, n_pages);
    const bool f16 = q_dtype == B2_F16;
    tree::launch_any(t, D, Hq, f16, pair, st);
    return launch_status("tree_attn");
  }
  p.ws = need ? (float*)workspace : nullptr;
  return attn::launch_simt(p, q_dtype, kv_dtype, st, "tree_attn");
}
