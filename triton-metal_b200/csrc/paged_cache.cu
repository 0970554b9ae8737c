// What a step does to a paged KV cache before attention reads it (sm_100a):
// the page table and the slot map from request lengths, and the new K/V rows
// written by slot.  The cache is the one decode_attn.cu reads: pages
// [n_pages, page_size, Hkv, D], page_table [B, max_pages] logical -> physical
// (paged_attention, triton_metal/codegen/_msl_templates.py:2279-2532; the
// reference fills both on the host and has no counterpart of these kernels).
#include "b2_common.cuh"
#include <type_traits>

namespace b2 {
namespace paged {

// ---------------------------------------------------------------------------
// build_page_table.  With c_b tokens in the cache and n_b new ones:
//   have_b = ceil(c_b / ps)              pages request b holds already
//   need_b = ceil((c_b + n_b) / ps) - have_b
//   token t of the step belongs to the request with off_b <= t < off_b + n_b
//   (off = exclusive sum of n), sits at pos = c_b + t - off_b, and its slot is
//   page * ps + pos % ps, where page is table[b, pos / ps] if pos / ps < have_b,
//   else free[base_b + pos / ps - have_b] (base = exclusive sum of need).
// A new page's first slot is always a new token's (pages fill from offset 0),
// so the thread of that token writes the table entry: every table entry is
// either read or written, never both, and nothing has to wait for anything.
// Latency sets the time (a step moves kilobytes), so it is one launch: every
// CTA redoes the scan over the requests up to its own tokens (kReqs of them
// per round) instead of waiting for a first kernel to publish it.  256 requests of
// one token: the kernel takes 4.2 us (calls in a graph; dependent loads: lengths,
// table or free list, slots), a call from Python 8.5, which is what the host needs
// for three outputs, their tuple and the launch; 93 prompts of up to 4099 tokens
// (1.6 MB) the same.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kPer = 4;                    // requests / tokens per thread
constexpr int kReqs = kThreads * kPer;     // requests per scan round
constexpr int kTokens = kThreads * kPer;   // tokens per CTA

struct TableParams {
  const int32_t *ctx, *fresh, *free_pages;
  int32_t* table;
  int64_t* slots;
  int32_t *offsets, *used;
  int64_t max_tokens, table_stride, n_free;
  int B, max_pages;
  uint32_t page_size;
};

// Tokens counted from 0 are at most 2 (2^31 - 1) here, so 32 unsigned bits hold
// them and their quotients (a 64-bit division costs several times as much).
__device__ __forceinline__ uint32_t pages_for(uint32_t tokens, uint32_t page_size) {
  return tokens / page_size + (tokens % page_size != 0);
}

__global__ void __launch_bounds__(kThreads) build_table_kernel(const TableParams p) {
  __shared__ int64_t sTok[kReqs + 1], sPage[kReqs];  // first token / first free page of each request
  __shared__ int32_t sCtx[kReqs];
  __shared__ int64_t wTok[kThreads / 32], wPage[kThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t t_lo = (int64_t)blockIdx.x * kTokens + tid * kPer;
  const int64_t cta_hi = min(p.max_tokens, (int64_t)(blockIdx.x + 1) * kTokens);
  const bool first = blockIdx.x == 0;
  if (first && tid == 0) p.offsets[0] = 0;
  int64_t tok0 = 0, page0 = 0;  // sums over the rounds before this one
  for (int r0 = 0; r0 < p.B; r0 += kReqs) {
    if (!first && tok0 >= cta_hi) break;  // CTA-uniform: later requests start behind this CTA's tokens
    int64_t n[kPer], g[kPer], ns = 0, gs = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = r0 + tid * kPer + e;
      uint32_t c = 0, m = 0;
      if (b < p.B) {
        c = max(p.ctx[b], 0);
        m = max(p.fresh[b], 0);
      }
      sCtx[tid * kPer + e] = (int32_t)c;
      n[e] = ns;
      g[e] = gs;
      ns += m;
      gs += pages_for(c + m, p.page_size) - pages_for(c, p.page_size);
    }
    int64_t ni = ns, gi = gs;  // inclusive scan over the warp, then over the warps
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, ni, off), b = __shfl_up_sync(0xffffffffu, gi, off);
      if (lane >= off) {
        ni += a;
        gi += b;
      }
    }
    if (lane == 31) {
      wTok[warp] = ni;
      wPage[warp] = gi;
    }
    __syncthreads();
    int64_t nb = tok0 + ni - ns, gb = page0 + gi - gs, nt = tok0, gt = page0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) {
        nb += wTok[w];
        gb += wPage[w];
      }
      nt += wTok[w];
      gt += wPage[w];
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = tid * kPer + e;
      sTok[i] = nb + n[e];
      sPage[i] = gb + g[e];
      if (first && r0 + i < p.B) p.offsets[r0 + i + 1] = (int32_t)(e + 1 < kPer ? nb + n[e + 1] : nb + ns);
    }
    if (tid == 0) sTok[kReqs] = nt;
    __syncthreads();
    // this thread's tokens that belong to the round's requests [tok0, nt)
    if (t_lo < nt && t_lo + kPer > tok0) {
      const int64_t ta = max(t_lo, tok0), tb = min(min(t_lo + kPer, nt), p.max_tokens);
      int lo = 0, hi = kReqs;  // sTok[lo] <= ta < sTok[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sTok[mid] <= ta) lo = mid;
        else hi = mid;
      }
      // where each token's page number stands, then all the loads together, then
      // the stores: one trip to memory for the kPer of them
      const int32_t* from[kPer];
      int32_t* entry[kPer];
      uint32_t off[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int64_t t = t_lo + e;
        from[e] = nullptr;
        entry[e] = nullptr;
        if (t < ta || t >= tb) continue;
        while (sTok[lo + 1] <= t) ++lo;
        const uint32_t c = sCtx[lo], pos = c + (uint32_t)(t - sTok[lo]), pi = pos / p.page_size;
        const uint32_t have = pages_for(c, p.page_size);
        off[e] = pos - pi * p.page_size;
        if (pi >= (uint32_t)p.max_pages) continue;
        int32_t* at = p.table + (int64_t)(r0 + lo) * p.table_stride + pi;
        if (pi < have) {
          from[e] = at;
        } else {
          const int64_t f = sPage[lo] + (pi - have);
          if (f < p.n_free) from[e] = p.free_pages + f;
          if (off[e] == 0) entry[e] = at;
        }
      }
      int64_t page[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) page[e] = from[e] ? *from[e] : -1;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (t_lo + e < ta || t_lo + e >= tb) continue;
        if (entry[e]) *entry[e] = (int32_t)page[e];
        p.slots[t_lo + e] = page[e] >= 0 ? page[e] * p.page_size + off[e] : -1;
      }
    }
    tok0 = nt;
    page0 = gt;
    __syncthreads();  // the arrays are rewritten by the next round
  }
  // room behind the last token
  for (int64_t t = max(t_lo, tok0); t < min(t_lo + kPer, p.max_tokens); ++t) p.slots[t] = -1;
  if (first && tid == 0) *p.used = (int32_t)page0;
}

// ---------------------------------------------------------------------------
// store_kv: row r of k / v (Hkv heads of D) goes to slot slots[r] of the
// pages; a slot outside [0, n_pages * page_size) is passed over.  A pure copy
// (or one rounding to the cache's type): 16-byte vectors of the cache's type,
// K and V of kRows rows in flight per thread.  Threads are laid out as
// (chunk of the row, row) with a power-of-two width, so that the division of
// a chunk by the head size is done once per thread and column, and the 64-bit
// division of a slot by the page size once per row (in shared memory).  60001
// fp32 rows of 8 x 128 into an fp16 cache, 738 MB: 131 us, 5.6 TB/s (0.86 of a
// copy's rate); 201 rows: 2.0 us in a graph, 5.2 a call.
// ---------------------------------------------------------------------------
constexpr int kMaxRows = 64;  // rows per CTA
constexpr int kRows = 4;      // rows in flight per thread

struct StoreParams {
  const void *k, *v;
  void *kp, *vp;
  const int64_t* slots;
  int64_t N, n_slots;
  int64_t ks[2], vs[2];      // (row, head) element strides
  int64_t kps[3], vps[3];    // (page, token, head)
  int page_size, chunks, head_chunks, width_log2, rows;  // chunks: vectors per row and per head
};

// VEC consecutive elements: loaded as TS, kept as TD
template <typename TS, typename TD, int VEC>
struct Chunk {
  TD d[VEC];
  __device__ __forceinline__ void load(const TS* p) {
    if constexpr (VEC == 1) {
      d[0] = conv(*p);
    } else if constexpr (std::is_same<TS, TD>::value) {
      *reinterpret_cast<uint4*>(d) = ld_stream_u4(p);
    } else {  // fp32 -> 16 bits: two 16-byte loads for one 16-byte store
      static_assert(sizeof(TS) == 4 && sizeof(TD) == 2 && VEC == 8, "fp32 to 16 bits");
      uint4 a = ld_stream_u4(p), b = ld_stream_u4(p + 4);
      const float f[8] = {__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w),
                          __uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w)};
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = from_f32<TD>(f[e]);
    }
  }
  static __device__ __forceinline__ TD conv(TS x) {
    if constexpr (std::is_same<TS, TD>::value) return x;
    else return from_f32<TD>(to_f32<TS>(x));
  }
  __device__ __forceinline__ void store(TD* p) const {
    if constexpr (VEC == 1) *p = d[0];
    else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(d);
  }
};

template <typename TS, typename TD, int VEC>
__global__ void __launch_bounds__(kThreads) store_kv_kernel(const StoreParams p) {
  __shared__ int64_t sK[kMaxRows], sV[kMaxRows];  // element offset of each row in the pages, -1 = passed over
  const int64_t row0 = (int64_t)blockIdx.x * p.rows;
  const int nr = (int)min((int64_t)p.rows, p.N - row0);
  for (int r = threadIdx.x; r < nr; r += kThreads) {
    const int64_t s = p.slots[row0 + r];
    int64_t ko = -1, vo = -1;
    if (s >= 0 && s < p.n_slots) {
      const int64_t pg = s / p.page_size, at = s - pg * p.page_size;
      ko = pg * p.kps[0] + at * p.kps[1];
      vo = pg * p.vps[0] + at * p.vps[1];
    }
    sK[r] = ko;
    sV[r] = vo;
  }
  __syncthreads();
  const int width = 1 << p.width_log2, tx = threadIdx.x & (width - 1), ty = threadIdx.x >> p.width_log2;
  const int nty = kThreads >> p.width_log2;
  for (int c = blockIdx.y * width + tx; c < p.chunks; c += gridDim.y * width) {
    const int h = c / p.head_chunks, d = (c - h * p.head_chunks) * VEC;
    const TS* k = (const TS*)p.k + row0 * p.ks[0] + h * p.ks[1] + d;
    const TS* v = (const TS*)p.v + row0 * p.vs[0] + h * p.vs[1] + d;
    TD* kp = (TD*)p.kp + h * p.kps[2] + d;
    TD* vp = (TD*)p.vp + h * p.vps[2] + d;
    for (int r0 = ty; r0 < nr; r0 += nty * kRows) {
      Chunk<TS, TD, VEC> a[kRows], b[kRows];
#pragma unroll
      for (int e = 0; e < kRows; ++e) {
        const int r = r0 + e * nty;
        if (r < nr && sK[r] >= 0) {
          a[e].load(k + r * p.ks[0]);
          b[e].load(v + r * p.vs[0]);
        }
      }
#pragma unroll
      for (int e = 0; e < kRows; ++e) {
        const int r = r0 + e * nty;
        if (r < nr && sK[r] >= 0) {
          a[e].store(kp + sK[r]);
          b[e].store(vp + sV[r]);
        }
      }
    }
  }
}

template <typename TS, typename TD, int VEC>
static void launch_store(StoreParams p, int64_t row_elems, int64_t D, cudaStream_t st) {
  p.chunks = (int)(row_elems / VEC);
  p.head_chunks = (int)(D / VEC);
  p.width_log2 = 0;
  while ((1 << p.width_log2) < p.chunks && (1 << p.width_log2) < kThreads) ++p.width_log2;
  // Rows per CTA: enough for kRows rows in flight a thread, fewer when that
  // would leave SMs without a CTA.
  const int64_t want = (int64_t)(kThreads >> p.width_log2) * kRows;
  const int64_t spread = (p.N + 2 * num_sms() - 1) / (2 * num_sms());
  int64_t rows = want < spread ? want : spread;
  if (rows > kMaxRows) rows = kMaxRows;
  p.rows = (int)(rows < 1 ? 1 : rows);
  const int64_t gx = (p.N + p.rows - 1) / p.rows;
  store_kv_kernel<TS, TD, VEC><<<dim3((unsigned)gx), kThreads, 0, st>>>(p);
}

}  // namespace paged
}  // namespace b2

using namespace b2;

extern "C" int b2_build_page_table(const int32_t* context_lens, const int32_t* new_lens, const int32_t* free_pages,
                                   int32_t* page_table, int64_t* slots, int32_t* offsets, int32_t* pages_used,
                                   int64_t B, int64_t page_size, int64_t n_free, int64_t max_pages,
                                   int64_t table_stride, int64_t max_tokens, void* stream) {
  B2_CHECK_ARG(B >= 0 && page_size > 0 && n_free >= 0 && max_pages >= 0 && max_tokens >= 0, B2_ERR_INVALID,
               "build_page_table: bad shape");
  B2_CHECK_ARG(B <= 2147483647 - paged::kReqs && page_size <= 2147483647 && max_pages <= 2147483647 &&
                   max_tokens <= 2147483647 - paged::kTokens,
               B2_ERR_INVALID, "build_page_table: sizes must stay below 2^31");
  B2_CHECK_ARG(table_stride >= max_pages, B2_ERR_INVALID, "build_page_table: table_stride %lld < max_pages %lld",
               (long long)table_stride, (long long)max_pages);
  B2_CHECK_ARG(offsets && pages_used && (!B || (context_lens && new_lens)) && (!max_tokens || slots) &&
                   (!n_free || free_pages) && (!B || !max_pages || page_table),
               B2_ERR_INVALID, "build_page_table: null pointer");
  paged::TableParams p;
  p.ctx = context_lens;
  p.fresh = new_lens;
  p.free_pages = free_pages;
  p.table = page_table;
  p.slots = slots;
  p.offsets = offsets;
  p.used = pages_used;
  p.max_tokens = max_tokens;
  p.table_stride = table_stride;
  p.n_free = n_free;
  p.B = (int)B;
  p.page_size = (uint32_t)page_size;
  p.max_pages = (int)max_pages;
  const int64_t grid = max_tokens ? (max_tokens + paged::kTokens - 1) / paged::kTokens : 1;
  paged::build_table_kernel<<<(unsigned)grid, paged::kThreads, 0, (cudaStream_t)stream>>>(p);
  return launch_status("build_page_table");
}

extern "C" int b2_store_kv(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots, int64_t N,
                           int64_t Hkv, int64_t D, int64_t n_pages, int64_t page_size, const int64_t* k_strides,
                           const int64_t* v_strides, const int64_t* kp_strides, const int64_t* vp_strides,
                           int src_dtype, int dst_dtype, void* stream) {
  B2_CHECK_ARG(N >= 0 && Hkv > 0 && D > 0 && n_pages >= 0 && page_size > 0, B2_ERR_INVALID, "store_kv: bad shape");
  B2_CHECK_ARG(page_size <= 2147483647 && N <= 2147483647 && Hkv <= 65535 && D <= 65535 && Hkv * D <= (1 << 24),
               B2_ERR_INVALID, "store_kv: sizes too large");
  B2_CHECK_ARG(k_strides && v_strides && kp_strides && vp_strides, B2_ERR_INVALID, "store_kv: null strides");
  const bool types = (src_dtype == dst_dtype && (dst_dtype == B2_F16 || dst_dtype == B2_BF16 || dst_dtype == B2_F32)) ||
                     (src_dtype == B2_F32 && (dst_dtype == B2_F16 || dst_dtype == B2_BF16));
  B2_CHECK_ARG(types, B2_ERR_DTYPE, "store_kv: rows of dtype %d into a cache of dtype %d", src_dtype, dst_dtype);
  if (N == 0 || n_pages == 0) return B2_OK;
  B2_CHECK_ARG(k && v && k_pages && v_pages && slots, B2_ERR_INVALID, "store_kv: null pointer");
  paged::StoreParams p;
  p.k = k;
  p.v = v;
  p.kp = k_pages;
  p.vp = v_pages;
  p.slots = slots;
  p.N = N;
  p.n_slots = n_pages * page_size;
  p.page_size = (int)page_size;
  const int es = src_dtype == B2_F32 ? 4 : 2, ed = dst_dtype == B2_F32 ? 4 : 2, vec = 16 / ed;
  bool wide = D % vec == 0 && aligned(k, 16) && aligned(v, 16) && aligned(k_pages, 16) && aligned(v_pages, 16);
  for (int i = 0; i < 2; ++i) {
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
    wide = wide && k_strides[i] * es % 16 == 0 && v_strides[i] * es % 16 == 0;
  }
  for (int i = 0; i < 3; ++i) {
    p.kps[i] = kp_strides[i];
    p.vps[i] = vp_strides[i];
    wide = wide && kp_strides[i] * ed % 16 == 0 && vp_strides[i] * ed % 16 == 0;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t row = Hkv * D;
  // 16-byte vectors where every row of every head starts on one, else one
  // element at a time
#define B2_STORE(TS, TD)                                                                                  \
  do {                                                                                                    \
    if (wide) paged::launch_store<TS, TD, 16 / (int)sizeof(TD)>(p, row, D, st);                           \
    else paged::launch_store<TS, TD, 1>(p, row, D, st);                                                   \
  } while (0)
  if (src_dtype == B2_F32 && dst_dtype == B2_F32) B2_STORE(float, float);
  else if (src_dtype == B2_F32 && dst_dtype == B2_F16) B2_STORE(float, __half);
  else if (src_dtype == B2_F32) B2_STORE(float, __nv_bfloat16);
  else if (src_dtype == B2_F16) B2_STORE(__half, __half);
  else B2_STORE(__nv_bfloat16, __nv_bfloat16);
#undef B2_STORE
  return launch_status("store_kv");
}
