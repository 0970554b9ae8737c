// Single tokens with capped or biased scores over a contiguous or paged cache
// (b2_decode_attn_scored, 16-bit): the drafted-tree kernel with one token a
// request, which shares the keys of all requests evenly among the SMs, whatever
// the requests' lengths.  (The plain decode kernel gives a (request, kv head) to
// one CTA; with lengths from 1 to 8192, 64 requests of 32 / 8 heads, its longest
// CTAs and the cap's two MUFU operations a score took 484 us where the cache is
// read in 164 us; this form takes 260 in pages of 16 keys, whose 2 KB boxes keep
// the copy engine busy that long, and 212 to 230 in larger ones.)
#include "tree_attn_kernel.cuh"

namespace b2 {
namespace tree {

// B2_ERR_UNSUPPORTED where this form does not take the call.
int launch_decode(const void* q, const void* k, const void* v, void* o, const int32_t* page_table,
                  const int32_t* seq_lens, void* workspace, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                  int64_t max_keys, int64_t page_size, int64_t max_pages, int64_t n_pages, const int64_t* k_strides,
                  const int64_t* v_strides, float scale, float softcap, const float* slopes, int dtype,
                  cudaStream_t st) {
  const int64_t rep = Hq / Hkv;
  bool wide = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(o, 16) && aligned(workspace, 16);
  for (int i = 0; i < 3; ++i) wide = wide && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0;
  if (!wide || dtype == B2_F32 || (D != 64 && D != 128) || rep > BR || !(scale > 0.f) || max_keys <= 0 || !workspace ||
      B > 65535 || max_keys > 2000000000 || Hkv * ((max_keys + BK - 1) / BK + kItemCost) > (1 << 30))
    return B2_ERR_UNSUPPORTED;
  Params t = {};
  t.q = (const uint16_t*)q;
  t.k = (const uint16_t*)k;
  t.v = (const uint16_t*)v;
  t.o = (uint16_t*)o;
  t.page_table = page_table;
  t.ctx = seq_lens;
  t.ws = (float*)workspace;
  t.n_pages = page_size ? n_pages : B;
  for (int i = 0; i < 3; ++i) {
    t.qs[i] = t.os[i] = i == 2 ? D : Hq * D;
    t.ks[i] = k_strides[i];
    t.vs[i] = v_strides[i];
  }
  t.B = (int)B;
  t.T = 1;
  t.Hkv = (int)Hkv;
  t.rep = (int)rep;
  t.cap = (int)max_keys;
  t.copies = copies_of(rep);
  t.tpt = (int)(BR / t.copies / rep);
  t.n_rt = 1;
  t.page_size = (uint32_t)page_size;
  t.max_pages = (int)max_pages;
  t.softcap = fa::make_cap(scale, softcap);
  t.slopes = slopes;
  t.err = device_error_word();
  t.box = box_of(page_size, n_pages);
  const bool f16 = dtype == B2_F16;
  if (!t.err) return B2_ERR_UNSUPPORTED;
  launch_any(t, D, Hq, f16, false, st);
  return launch_status("decode_attn_scored");
}

}  // namespace tree
}  // namespace b2
