// What the attention kernels with score forms and row masks share: the key
// range of a prompt's row, the score forms, and the parameters of the
// CUDA-core kernel (attn_simt.cu).
#pragma once
#include "b2_common.cuh"

namespace b2 {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// Keys a prompt's query row sees: one range [lo, hi) for every kind of mask.
//   causal      hi = row + 1; a window raises lo to row + 1 - window
//   doc_offsets int32 [B, n_docs + 1], ascending: rows and keys off[d] ..
//               off[d+1] - 1 are document d and see only their document; a row
//               in no document sees nothing
//   prefix      int32 [B, max(n_docs, 1)]: the first prefix tokens of a
//               document (without documents: of the prompt) are seen by all
//               of its rows
struct RangeMask {
  int causal, window, n_docs;
  const int32_t *docs, *prefix;
};

__device__ __forceinline__ void row_range(const RangeMask& m, int b, int row, int Skv, int& lo, int& hi) {
  lo = 0;
  hi = Skv;
  int d = 0, start = 0;  // document and its first token, which may lie before the row's
  if (m.docs) {
    const int32_t* off = m.docs + (int64_t)b * (m.n_docs + 1);
    int a = 0, z = m.n_docs;  // d = how many of off[1..n_docs] are <= row
    while (a < z) {
      const int mid = (a + z) >> 1;
      if (off[mid + 1] <= row) a = mid + 1;
      else z = mid;
    }
    d = a;
    lo = hi = 0;
    if (d < m.n_docs && off[d] <= row && row < off[d + 1]) {
      start = off[d];
      lo = max(start, 0);
      hi = min(off[d + 1], Skv);
    }
  }
  if (m.causal) {
    int last = row + 1;
    if (m.prefix) {
      // prefix lengths are clamped so that the sum stays in 32 bits
      const int p = m.prefix[(int64_t)b * max(m.n_docs, 1) + min(d, max(m.n_docs, 1) - 1)];
      last = max(last, start + (start < 0 ? max(p, 0) : min(max(p, 0), Skv)));
    }
    hi = min(hi, last);
    if (m.window > 0) lo = max(lo, row - m.window + 1);
  }
  hi = max(hi, lo);
}

// tanh to about 2e-7: an odd Taylor series below 0.35 (its next term there is
// under 1e-8), (1 - t) / (1 + t) with t = e^-2|x| above.  (The one-instruction
// tanh is good to 2^-11, which a cap of 50 turns into 0.02 in the exponent.)
__device__ __forceinline__ float tanh_acc(float x) {
  const float ax = fabsf(x), x2 = x * x;
  float s = -0.0088632356f;                      // -1382/155925
  s = fmaf(s, x2, 0.021869489f);                 // 62/2835
  s = fmaf(s, x2, -0.053968254f);                // -17/315
  s = fmaf(s, x2, 0.13333333f);
  s = fmaf(s, x2, -0.33333333f);
  const float small = fmaf(x * x2, s, x);
  const float t = __expf(-2.f * ax);
  const float big = copysignf(__fdividef(1.f - t, 1.f + t), x);
  return ax < 0.35f ? small : big;
}

// A cap beyond these bounds gives the same weights in fp32 (equal ones below, the
// uncapped scores' above), but its products would leave fp32's range.
inline float cap_in_range(float cap) { return cap > 0.f ? (cap < 1e-30f ? 1e-30f : cap > 1e30f ? 1e30f : cap) : cap; }

// Parameters of the CUDA-core kernel.  Rows of one (batch b, kv head hk) are
// r = s * rep + hh (query position s, query head hk * rep + hh).
struct SimtParams {
  const void *q, *k, *v;
  void* o;
  int B, T, Hq, Hkv, D, Skv;                 // T query positions; Skv: keys a sequence may reach
  int64_t qs[3], os[3];                      // (b, s, h) element strides
  int64_t ks[3], vs[3];                      // contiguous (b, h, s); paged (page, token, head)
  const int32_t* page_table;                 // paged: [B, max_pages]
  int page_size, max_pages;
  int64_t n_pages;
  float scale, softcap;                      // softcap 0: none
  const float* slopes;                       // [Hq] or null
  RangeMask range;                           // used when tree_mask is null
  const uint8_t* tree_mask;                  // [B or 1, T, T], non-zero: row sees drafted token
  int64_t tree_stride;                       // 0 or T * T
  const int32_t *ctx, *draft;                // tree: context / draft lengths (draft null: T)
  float* ws;                                 // split partials, rows of (m, l, D values)
  int nsplit, split_len;
  int wide;                                  // set by launch_simt: 16-byte loads of K / V rows
  unsigned* err;
};

// Keys and drafted tokens of sequence b of a tree, within the cache.
__device__ __forceinline__ void tree_lens(const int32_t* ctx, const int32_t* draft, int b, int T, int cap, int& c,
                                          int& dl) {
  c = min(max(ctx[b], 0), cap);
  dl = draft ? min(max(draft[b], 0), T) : T;
  dl = min(dl, cap - c);
}

// Error codes of the device error word (b2_device_error)
constexpr unsigned kErrPage = 0xB2500001u;  // a page table entry outside of the cache

int simt_splits(int64_t row_tiles, int64_t max_keys);
int launch_simt(SimtParams p, int q_dtype, int kv_dtype, cudaStream_t st, const char* what);
size_t simt_workspace(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_keys);

}  // namespace attn
}  // namespace b2
