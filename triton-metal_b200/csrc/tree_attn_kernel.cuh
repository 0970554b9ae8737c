// Attention of a tree of drafted tokens over a contiguous or paged KV cache
// (speculative decoding), sm_100a.
//
//   s = scale q.k  (softcap: s = cap tanh(s / cap)),  o = softmax(s | mask) v
//
// The rows of one (request, kv head) are its T drafted tokens times the
// Hq / Hkv query heads: row r = t * rep + hh.  Each K/V row is needed by all of
// them, so the cache is the traffic: with D = 128 and 16-bit values a key costs
// 512 bytes and 512 FLOPs a row, which meets the HBM rate at ~250 rows.  Up to
// there the copy stream sets the time, and the tensor cores have to keep up
// with it at any number of rows, which 128-row tcgen05 tiles do.
//
// One persistent CTA per SM.  Work is cut in 128-key tiles; the tiles of all
// (request, kv head, row tile) items stand in one line and every CTA takes an
// equal run of it, whatever the requests' lengths (they are on the GPU only).
// A run is a few segments, each inside one item; a segment that is not a whole
// item leaves (m, l, unnormalised o) in the workspace, and a second kernel
// joins those.
// TMA form (contiguous caches, and page sizes that are a multiple of 8 keys):
//   warp 0      TMA for Q, K and V into a ring of kRing tiles, in the order
//               K0 K1 V0 K2 V1 ...; a box is as many keys as divide a page and a
//               tile.  Pages of 16 keys need eight boxes of 2 KB for 16 KB; with
//               V copied by two warps instead, so that the copy engine had half
//               the boxes, single tokens of 64 requests (32 / 8 heads of 128, up to
//               8192 keys, cap and bias) took 365 us, not 282.
//   warp 1      TMEM owner and MMA issuer
//   warps 2-3   pass the tiles on; in V tiles with drafted tokens they zero the
//               rows behind the last key and what is infinite or NaN
//   warps 4-11  two softmax warpgroups, one row per thread (TMEM lane = row)
// cp.async form (other page sizes, and tensors that no tensor map describes):
// warps 0-2 copy with 16-byte cp.async and do the zeroing, warp 3 issues the MMAs.
// TMEM as in the prefill kernel: unit u has S_u / P_u at column 256u and O_u at
// 256u + 128.  With one row tile per item (SINGLE) the two units take the even
// and the odd key tiles of the same rows, so that one unit's softmax runs under
// the other's MMAs, and their (m, l, O) are joined from TMEM at the segment's
// end; with more row tiles (PAIR) the units are two row tiles that share every
// K/V tile.
// Few rows (at most 64 or 32) would leave most softmax warps idle, since a warp
// reaches only its own 32 TMEM lanes: such rows stand in the tile 2 or 4 times,
// and each copy takes every 2nd or 4th part of a tile's keys (its P is 0 for the
// others), so that all warps share the exponentials.  The copies are joined like
// the units, through shared memory.
// Measured: trees of 64, 32 requests of 8 to 32 thousand keys, 32 / 8 heads of
// 128, bf16: 0.86 to 0.91 ms, 3.1 TB/s and 770 TF/s (either floor is 0.42 ms);
// trees of 26, 16 requests of up to 4096 keys in pages of 16, fp16: 57 us, 2.5 TB/s
// (starts and ends of segments); a tree of 8, one request of 500 keys: 19 to 20 us
// (two launches and one chain).
#pragma once
#include "attn_common.cuh"
#include "fa_common.cuh"
#include <math.h>

namespace b2 {
namespace tree {

using namespace fa;

constexpr int kThreads = 384;
constexpr int kCopyRows = 44;              // cp.async form: rows of a copying warp (the third: 40)
constexpr int BR = 128, BK = 128;          // rows and keys of a tile
// What starting and ending an item costs, in tiles (0 instead of 2: trees of 26
// over 16 requests 67 us, not 56; single tokens of 64 requests 307 us, not 260).
constexpr int kItemCost = 2;

template <int HD>
struct Cfg {
  static constexpr int kAtom = 128 * 128;             // 128 rows x 128 bytes
  static constexpr int kTile = HD / 64 * kAtom;
  static constexpr int kRing = HD == 128 ? 5 : 10;    // 160 KB of K and V tiles
  // tiles a copying thread leaves in flight behind the one it hands over
  static constexpr int kLag = HD == 128 ? 2 : 4;
  static constexpr int kHead = 3 * 1024;                 // barriers and the (m, l) exchange
  static constexpr int kSmem = kHead + (2 + kRing) * kTile;
  static_assert(kSmem <= 232448, "shared memory");
  static_assert(kLag < kRing, "a ring slot is handed over before it is waited for again");
};

struct Params {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  const int32_t *page_table, *ctx, *draft;
  const uint8_t* mask;
  float* ws;
  int64_t mask_stride, n_pages;
  int64_t qs[3], os[3], ks[3], vs[3];
  int B, T, Hkv, rep, cap;      // rep: query heads of a kv head; cap: keys a cache row holds
  int tpt;                      // drafted tokens of a row tile, rows t * rep + head
  int copies;                   // how often the rows stand in the tile (SINGLE: 1, 2 or 4)
  int n_rt;                     // items of a kv head: row tiles (PAIR: pairs of them)
  uint32_t page_size;           // 0: contiguous
  int max_pages;
  int box;                      // TMA: keys of a K / V box
  Cap softcap;
  const float* slopes;          // BIAS: [Hq]
  unsigned* err;
};

// ------------------------------------------------------------- schedule
// Items of request b: hk-major, then row tile.  A row tile with drafted tokens
// has all of the request's key tiles, one without has a single tile in which
// nothing is visible (its rows become 0).  The line that the CTAs share is made
// of units: kItemCost units that stand for an item's start and end, then its
// tiles.
struct Req {
  int ctx, dl, tiles, full;  // key tiles, row tiles with drafted tokens
  int per_head;              // units of one kv head
};
__device__ __forceinline__ Req request(const Params& p, int b, int tokens) {
  Req r;
  if (p.mask) {
    attn::tree_lens(p.ctx, p.draft, b, p.T, p.cap, r.ctx, r.dl);
  } else {  // single tokens: ctx holds sequence lengths, the last key is the token's own
    const int n = min(max(p.ctx[b], 0), p.cap);
    r.dl = n > 0;
    r.ctx = n - r.dl;
  }
  r.tiles = (r.ctx + r.dl + BK - 1) / BK;
  r.full = (r.dl + tokens - 1) / tokens;
  r.per_head = r.full * (r.tiles + kItemCost) + (p.n_rt - r.full) * (1 + kItemCost);
  return r;
}

struct Segment {
  int b, hk, rt, tile, n, of;  // n tiles from `tile` on, of an item with `of` tiles
  int ctx, dl, keys;           // keys = ctx + dl, 0 when the item has no drafted token
};

// Walks the segments of the run [g, g1) of units.
struct Walk {
  int64_t g, g1, start;  // start: first unit of request b
  int b;
  Req r;
  __device__ __forceinline__ bool next(const Params& p, int tokens, Segment& s) {
    while (g < g1) {
      while (g >= start + (int64_t)r.per_head * p.Hkv) {
        start += (int64_t)r.per_head * p.Hkv;
        r = request(p, ++b, tokens);
      }
      const uint32_t local = (uint32_t)(g - start);
      s.b = b;
      s.hk = local / (uint32_t)r.per_head;
      int rem = local - (uint32_t)s.hk * r.per_head;
      const int size = r.tiles + kItemCost;
      const bool has = rem < r.full * size;
      if (!has) rem -= r.full * size;
      s.of = has ? r.tiles : 1;
      s.rt = rem / (s.of + kItemCost);
      const int at = rem - s.rt * (s.of + kItemCost);  // unit within the item
      if (!has) s.rt += r.full;
      const int end = (int)min((int64_t)(s.of + kItemCost), at + (g1 - g));
      s.tile = max(at - kItemCost, 0);
      s.n = max(end - kItemCost, 0) - s.tile;
      s.ctx = r.ctx;
      s.dl = has ? r.dl : 0;
      s.keys = has ? r.ctx + r.dl : 0;
      g += end - at;
      if (s.n > 0) return true;  // else the run ends before the item's first tile
    }
    return false;
  }
};

// First unit of CTA c's run when G CTAs share W units (G <= W, so that no run
// is empty).
__device__ __forceinline__ int64_t run_start(int64_t c, int64_t W, int64_t G) {
  const int64_t n = c * W;
  return n >> 32 == 0 ? (uint32_t)n / (uint32_t)G : n / G;
}

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int off = 16; off; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// ------------------------------------------------------------- masks
// Drafted tokens j0 .. j0 + 127 that this thread's row sees, as bits.  The warp
// reads the mask rows of its tokens t0 .. t1 together (lane = drafted token),
// eight rows in flight, and every lane keeps the ballots of its own token t.
__device__ __forceinline__ void draft_bits(uint32_t (&bits)[4], const uint8_t* mask, int T, int t, int t0, int t1,
                                           int j0, int dl) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 0; w < 4; ++w) bits[w] = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int j = j0 + 32 * w + lane;
    if (j0 + 32 * w >= dl) break;  // the same for the warp
    for (int tt = t0; tt <= t1; tt += 8) {
      bool see[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) see[i] = j >= 0 && j < dl && tt + i <= t1 && (!mask || mask[(int64_t)(tt + i) * T + j] != 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = __ballot_sync(0xffffffffu, see[i]);
        if (tt + i == t) bits[w] = b;
      }
    }
  }
}

// Visible keys among the 128 from drafted token j0 (negative: context) on, from
// the bits of the first 128 drafted tokens.  
__device__ __forceinline__ void visible_bits(uint32_t (&vis)[4], const uint32_t (&bits)[4], int j0) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int j = j0 + 32 * w;
    uint32_t x;
    if (j <= -32) {
      x = 0xffffffffu;
    } else if (j < 0) {
      x = ((1u << -j) - 1) | bits[0] << -j;
    } else {
      const int i = j >> 5;
      const uint32_t lo = i == 0 ? bits[0] : i == 1 ? bits[1] : i == 2 ? bits[2] : i == 3 ? bits[3] : 0;
      const uint32_t hi = i == 0 ? bits[1] : i == 1 ? bits[2] : i == 2 ? bits[3] : 0;
      x = __funnelshift_r(lo, hi, j & 31);
    }
    vis[w] = x;
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// any_of_softmax of one softmax warpgroup
__device__ __forceinline__ bool any_of_warpgroup(int u, bool x) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %2, 0;\n barrier.cta.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(3 + u), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void warpgroup_sync(int u) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(3 + u) : "memory"); }
__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 2, 256;" ::: "memory"); }

// Page table entry of key `pos` of request b (contiguous: 0).
__device__ __forceinline__ int key_page(const Params& p, int b, int pos) {
  return p.page_size ? p.page_table[(int64_t)b * p.max_pages + (uint32_t)pos / p.page_size] : 0;
}

// Element offset of key `pos` of request b and kv head hk in K or V, given its
// page; false when that is none of the cache's.
__device__ __forceinline__ bool key_offset(const Params& p, int b, int hk, int pos, int pg, int64_t& ko, int64_t& vo) {
  if (p.page_size) {
    const uint32_t at = (uint32_t)pos % p.page_size;
    ko = pg * p.ks[0] + at * p.ks[1] + hk * p.ks[2];
    vo = pg * p.vs[0] + at * p.vs[1] + hk * p.vs[2];
    return pg >= 0 && pg < p.n_pages;
  }
  ko = b * p.ks[0] + hk * p.ks[1] + (int64_t)pos * p.ks[2];
  vo = b * p.vs[0] + hk * p.vs[1] + (int64_t)pos * p.vs[2];
  return true;
}

// ring index of K_i and V_i within a segment of n tiles: K0 K1 V0 K2 V1 ... V(n-1)
__device__ __forceinline__ int k_at(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int v_at(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

template <int HD, int FMT, bool PAIR, bool CAP, bool BIAS, bool TMA>
__global__ void __launch_bounds__(kThreads, 1)
tree_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
            const __grid_constant__ CUtensorMap tmV, const Params p) {
  using C = Cfg<HD>;
  constexpr int NS = C::kRing, LAG = C::kLag, NT = kThreads, kMmaWarp = TMA ? 1 : 3;
  constexpr int kRows = PAIR ? 2 * BR : BR;  // rows of an item
  const int tokens = p.tpt * (PAIR ? 2 : 1), br = p.tpt * p.rep;  // of an item; rows of a tile
  const int copies = PAIR ? 1 : p.copies, rw = BR / copies;       // rows a copy takes up
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_raw);
  uint64_t* ready = full + NS;        // TMA: a tile passed on by warps 2-3 (else unused)
  uint64_t* empty = ready + NS;
  uint64_t* s_full = empty + NS;      // [2]
  uint64_t* p_ready = s_full + 2;     // [2]
  uint64_t* o_done = p_ready + 2;     // [2]
  uint64_t* epi_done = o_done + 2;    // [2] by segment parity
  uint64_t* drain = epi_done + 2;
  int64_t* s_run = reinterpret_cast<int64_t*>(drain + 1);    // [16] scan of the schedule
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(s_run + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile uint32_t* s_bad = reinterpret_cast<volatile uint32_t*>(tmem_holder + 2);  // [2] by segment parity
  int* s_b = reinterpret_cast<int*>(tmem_holder + 4);
  float2* s_ml = reinterpret_cast<float2*>(smem_raw + 512);  // [2][128]
  static_assert((3 * NS + 9 + 16) * 8 + 5 * 4 <= 512 && 512 + 2 * 128 * 8 <= C::kHead - 512, "header");
  // tiles start on the next 1024-byte boundary behind the header
  const uint32_t pad = (1024 - ((raw + 2560) & 1023)) & 1023;
  uint8_t* sQ = smem_raw + 2560 + pad;  // 2 tiles: PAIR both row tiles, else this and the next segment's
  uint8_t* sRing = sQ + 2 * C::kTile;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // the joining kernel may start (it waits for this one's end)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], TMA ? 1 : 96);
      mbar_init(&ready[i], 2);
      mbar_init(&empty[i], 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&s_full[u], 1);
      mbar_init(&p_ready[u], 4);
      mbar_init(&o_done[u], 1);
      mbar_init(&epi_done[u], 8);
      s_bad[u] = 0xffffffffu;
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(tmem_holder, 512);
    tc::tmem_relinquish();
  }
  // this CTA's run, and the request that its first unit is in: a scan over the
  // requests' units, in rounds of one request a thread
  int64_t mine = 0;
  if (tid < p.B) mine = (int64_t)request(p, tid, tokens).per_head * p.Hkv;
  auto scan = [&](int64_t x, int64_t& total) {  // sum over the threads before this one
    int64_t inc = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += a;
    }
    __syncthreads();  // s_run of the round before is read
    if (lane == 31) s_run[warp] = inc;
    __syncthreads();
    int64_t before = inc - x;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) before += s_run[w];
      total += s_run[w];
    }
    return before;
  };
  tc::fence_before_sync();
  int64_t round = 0, start = scan(mine, round), W = round;
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  for (int b0 = NT; b0 < p.B; b0 += NT) {
    int64_t t;
    scan(b0 + tid < p.B ? (int64_t)request(p, b0 + tid, tokens).per_head * p.Hkv : 0, t);
    W += t;
  }
  const int64_t G = min((int64_t)gridDim.x, W);
  Walk walk;
  walk.g = walk.g1 = 0;
  if (blockIdx.x < G) {
    walk.g = run_start(blockIdx.x, W, G);
    walk.g1 = run_start(blockIdx.x + 1, W, G);
  }
  bool fits = 2560 + pad + (2 + NS) * C::kTile <= (uint32_t)C::kSmem;
  if (!fits && tid == 0) atomicCAS(p.err, 0u, 0xB2400001u);
  const bool some = walk.g < walk.g1 && fits;
  if (some) {
    int64_t before = 0;  // units of the rounds before
    for (int b0 = 0;; b0 += NT) {
      if (b0) {
        mine = b0 + tid < p.B ? (int64_t)request(p, b0 + tid, tokens).per_head * p.Hkv : 0;
        start = before + scan(mine, round);
      }
      if (start <= walk.g && walk.g < start + mine) {
        *s_b = b0 + tid;
        s_run[15] = start;
      }
      before += round;
      if (before > walk.g) break;  // the same for every thread
    }
    __syncthreads();
    walk.b = *s_b;
    walk.start = s_run[15];
    walk.r = request(p, walk.b, tokens);
  }

  Segment sg;
  // key tile that the segment's i-th turn takes: with a bias from the last one on
  auto key_tile = [&](int i) { return sg.tile + (BIAS ? sg.n - 1 - i : i); };
  if (TMA && some && warp == 0) {
    // ----------------------------------- TMA -----------------------------------
    // Lane i issues box i / NA, columns 64 (i % NA).
    constexpr int NA = HD / 64;
    const int boxes = BK / p.box, mine_box = lane / NA, atom = lane % NA;
    const bool has_box = mine_box < boxes;
    uint32_t seq = 0, seg = 0;
    bool ok = true;
    auto load4 = [&](uint8_t* dst, const CUtensorMap* m, int c1, int c2, int c3, uint64_t* bar) {
      tma_load_4d(dst, m, atom * 64, c1, c2, c3, bar);
    };
    // K or V tile `tile` of the segment (this lane's page: pg), with Q when that
    // rides along (q_tiles)
    auto issue = [&](const CUtensorMap* m, int tile, int pg, int q_tiles) {
      const uint32_t slot = seq % NS;
      ok = __all_sync(0xffffffffu, wait_abort(&empty[slot], ((seq / NS) & 1) ^ 1, p.err, 0xB2400002u, abort_flag));
      if (!ok) return;
      uint8_t* dst = sRing + slot * C::kTile + atom * C::kAtom + mine_box * p.box * 128;
      const int pos = key_tile(tile) * BK + mine_box * p.box;
      bool valid = has_box && pos < sg.keys;
      if (valid && p.page_size && (pg < 0 || pg >= p.n_pages)) {
        valid = false;  // none of the cache's pages: zeros
        atomicCAS(p.err, 0u, attn::kErrPage);
        for (int i = 0; i < p.box * 8; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
        tc::fence_proxy_async_smem();
      }
      const int n = __popc(__ballot_sync(0xffffffffu, valid));
      __syncwarp();  // zeros written before the arrival that hands them over
      if (lane == 0) mbar_arrive_expect_tx(&full[slot], n * p.box * 128 + q_tiles * copies * NA * br * 128);
      __syncwarp();
      if (valid) {
        if (p.page_size) load4(dst, m, sg.hk, (uint32_t)pos % p.page_size, pg, &full[slot]);
        else load4(dst, m, pos, sg.hk, sg.b, &full[slot]);
      }
      if (lane < q_tiles * copies * NA) {
        const int i = lane / NA, rt = PAIR ? 2 * sg.rt + i : sg.rt;  // PAIR: row tile, else copy
        load4(sQ + (PAIR ? i : seg & 1) * C::kTile + atom * C::kAtom + (PAIR ? 0 : i * rw * 128), &tmQ, sg.hk * p.rep,
              rt * p.tpt, sg.b, &full[slot]);
      }
      ++seq;
    };
    while (ok && walk.next(p, tokens, sg)) {
      auto page = [&](int tile) {
        const int pos = key_tile(tile) * BK + mine_box * p.box;
        return has_box && tile < sg.n && pos < sg.keys ? key_page(p, sg.b, pos) : 0;
      };
      int pg = page(0), pg1 = page(1);  // one tile ahead
      if (PAIR ? seg >= 1 : seg >= 2) {
        // Q of the segment before (PAIR) or of the one before that is free once
        // its epilogue is over
        const uint32_t prev = seg - (PAIR ? 1 : 2);
        ok = __all_sync(0xffffffffu, wait_abort(&epi_done[prev & 1], (prev >> 1) & 1, p.err, 0xB2400003u, abort_flag));
        if (!ok) break;
      }
      const int q_tiles = PAIR && (2 * sg.rt + 1) * p.tpt < p.T ? 2 : 1;
      issue(&tmK, 0, pg, q_tiles);
      for (int i = 0; i < sg.n && ok; ++i) {
        const int pg2 = page(i + 2);
        if (i + 1 < sg.n) issue(&tmK, i + 1, pg1, 0);
        if (ok) issue(&tmV, i, pg, 0);
        pg = pg1;
        pg1 = pg2;
      }
      ++seg;
    }
  } else if (TMA && some && (warp == 2 || warp == 3)) {
    // ---------------------------- tiles passed on ----------------------------
    // Behind the last key a page holds what was there before; a drafted token's
    // V that is infinite or NaN must reach only the rows that see the token.  In
    // P V a weight of 0 would make NaN of both: the former is zeroed, the latter
    // zeroed and added for those rows at the segment's end.
    uint32_t seq = 0, seg = 0;
    bool ok = true;
    while (ok && walk.next(p, tokens, sg)) {
      for (int e = 0; e < 2 * sg.n; ++e, ++seq) {
        const uint32_t slot = seq % NS;
        ok = __all_sync(0xffffffffu, wait_abort(&full[slot], (seq / NS) & 1, p.err, 0xB240000Bu, abort_flag));
        if (!ok) break;
        const int i = e == 2 * sg.n - 1 ? sg.n - 1 : e > 0 && e % 2 == 0 ? e / 2 - 1 : -1;  // V_i, or -1: a K tile
        const int kv0 = key_tile(i) * BK;
        if (i >= 0 && kv0 + BK > sg.ctx) {
          uint4* tile = reinterpret_cast<uint4*>(sRing + slot * C::kTile);
          const int first = max(sg.ctx - kv0, 0), last = sg.keys - kv0;  // drafted rows, then rows behind the end
          bool bad = false;
          for (int x = tid - 64 + first * 8; x < 128 * 8 * (HD / 64); x += 64) {
            const int row = x / 8 % 128;
            if (row < first) continue;
            uint4 val = tile[x];
            if (row >= last) {
              tile[x] = make_uint4(0, 0, 0, 0);
            } else if (zero_not_finite<FMT>(val)) {
              tile[x] = val;
              bad = true;
            }
          }
          // tagged with the segment, so that nobody has to clear it
          if (bad) s_bad[seg & 1] = seg;
          tc::fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ready[slot]);
      }
      ++seg;
    }
  }
  if (!TMA && some && warp < 3) {
    // --------------------------------- copies ---------------------------------
    constexpr int CH = HD / 8, RPP = 32 / CH;  // 16-byte chunks of a row, rows a warp copies at once
    const int cc = lane % CH, rsub = lane / CH;
    const int row0 = kCopyRows * warp, its = (warp == 2 ? 128 - 2 * kCopyRows : kCopyRows) / RPP;
    uint32_t seq = 0, handed = 0;  // tiles issued / handed over
    uint32_t end0 = 0, end1 = 0;   // seq at the end of the last segment and of the one before
    uint64_t meta = 0;             // 12 bits a tile in flight: first drafted row of a V tile (255: none), parity
    bool ok = true;
    auto chunk_at = [&](uint32_t tile, int r) {
      return tile + (cc >> 3) * C::kAtom + r * 128 + (((cc & 7) ^ (r & 7)) << 4);
    };
    uint32_t seg = 0;
    // A drafted token's V that is infinite or NaN must reach only the rows that
    // see the token, but in P V a weight of 0 would make NaN of it: such values
    // are zeroed here and added for those rows at the segment's end.
    auto hand_over = [&](uint32_t m) {
      const uint32_t slot = handed % NS;
      const int first = m & 255;
      if (first < 128) {
        bool bad = false;
        const uint32_t tile = smem_u32(sRing) + slot * C::kTile;
        for (int i = 0; i < its; ++i) {
          const int r = row0 + RPP * i + rsub;
          if (r < first) continue;
          uint4* at = reinterpret_cast<uint4*>(sRing + (chunk_at(tile, r) - smem_u32(sRing)));
          uint4 x = *at;
          const bool hit = zero_not_finite<FMT>(x);
          if (hit) *at = x;
          bad |= hit;
        }
        // tagged with the segment, so that nobody has to clear it
        if (bad) s_bad[(m >> 8) & 1] = seg - ((seg & 1) != ((m >> 8) & 1));
      }
      tc::fence_proxy_async_smem();
      mbar_arrive(&full[slot]);
      ++handed;
    };
    auto begin = [&]() {  // the slot of the next tile, once it is free
      const uint32_t slot = seq % NS;
      ok = __all_sync(0xffffffffu, wait_abort(&empty[slot], ((seq / NS) & 1) ^ 1, p.err, 0xB2400002u, abort_flag));
      return smem_u32(sRing) + slot * C::kTile;
    };
    auto end = [&](uint32_t m) {
      cp_async_commit();
      meta = meta << 12 | m;
      ++seq;
      if (seq - handed > LAG) {
        cp_async_wait<LAG>();
        hand_over((uint32_t)(meta >> (12 * LAG)) & 0xfff);
      }
    };
    auto drain_all = [&]() {
      cp_async_wait<0>();
      while (handed != seq) hand_over((uint32_t)(meta >> (12 * (seq - handed - 1))) & 0xfff);
    };
    // element offsets of this warp's rows: lane i has rows i and 32 + i; < 0: zeros
    struct Rows {
      int64_t a, b;
    };
    auto copy_tile = [&](uint32_t tile, const uint16_t* base, const Rows& off) {
#pragma unroll
      for (int i = 0; i < kCopyRows / RPP; ++i) {
        if (i >= its) break;
        const int64_t o = __shfl_sync(0xffffffffu, RPP * i < 32 ? off.a : off.b, (RPP * i + rsub) & 31);
        const int r = row0 + RPP * i + rsub;
        cp_async16(chunk_at(tile, r), base + (o < 0 ? 0 : o) + cc * 8, o >= 0);
      }
    };
    while (ok && walk.next(p, tokens, sg)) {
      if (PAIR ? seg >= 1 : seg >= 2) {
        // Q of the segment before (PAIR) or of the one before that is free once
        // its epilogue is over; that waits for its last tile, which must not be
        // among those still to be handed over
        if (handed < (PAIR ? end0 : end1)) drain_all();
        const uint32_t prev = seg - (PAIR ? 1 : 2);
        ok = __all_sync(0xffffffffu,
                        wait_abort(&epi_done[prev & 1], (prev >> 1) & 1, p.err, 0xB2400003u, abort_flag));
        if (!ok) break;
      }
      // this lane's keys of each tile, one tile ahead, and their pages, two ahead
      Rows ko, vo, ko1 = {-1, -1}, vo1 = {-1, -1};
      auto key = [&](int tile, int half) {  // -1: none
        const int at = 32 * half + lane, pos = key_tile(tile) * BK + row0 + at;
        return tile < sg.n && at < kCopyRows && row0 + at < BK && pos < sg.keys ? pos : -1;
      };
      auto page = [&](int tile) {
        const int a = key(tile, 0), b = key(tile, 1);
        return make_int2(a < 0 ? 0 : key_page(p, sg.b, a), b < 0 ? 0 : key_page(p, sg.b, b));
      };
      auto locate = [&](int tile, int2 pg, Rows& k, Rows& v) {
        const int a = key(tile, 0), b = key(tile, 1);
        k = {-1, -1};
        v = {-1, -1};
        bool fine = true;
        if (a >= 0 && !key_offset(p, sg.b, sg.hk, a, pg.x, k.a, v.a)) k.a = v.a = -1, fine = false;
        if (b >= 0 && !key_offset(p, sg.b, sg.hk, b, pg.y, k.b, v.b)) k.b = v.b = -1, fine = false;
        if (!fine) atomicCAS(p.err, 0u, attn::kErrPage);
      };
      const int2 pg0 = page(0);
      int2 pg1 = page(1);
      locate(0, pg0, ko, vo);
      uint32_t tile = begin();
      if (!ok) break;
#pragma unroll 1
      for (int u = 0; u < (PAIR ? 2 : 1); ++u) {
        const int rt = PAIR ? 2 * sg.rt + u : sg.rt;
        auto q_row = [&](int at) {
          const int row = (row0 + at) & (rw - 1), t = rt * p.tpt + row / p.rep;
          return at < kCopyRows && row < br && t < p.T
                     ? sg.b * p.qs[0] + (int64_t)t * p.qs[1] + (int64_t)(sg.hk * p.rep + row % p.rep) * p.qs[2]
                     : (int64_t)-1;
        };
        const Rows off = {q_row(lane), q_row(32 + lane)};
        copy_tile(smem_u32(sQ) + (PAIR ? u : seg & 1) * C::kTile, p.q, off);
      }
      copy_tile(tile, p.k, ko);
      end(255);
      for (int i = 0; i < sg.n && ok; ++i) {
        if (i + 1 < sg.n) {
          locate(i + 1, pg1, ko1, vo1);
          pg1 = page(i + 2);
          tile = begin();
          if (!ok) break;
          copy_tile(tile, p.k, ko1);
          end(255);
        }
        tile = begin();
        if (!ok) break;
        copy_tile(tile, p.v, vo);
        const int first = max(sg.ctx - key_tile(i) * BK, 0);
        end((first < 128 && sg.dl > 0 ? first : 255) | (seg & 1) << 8);
        vo = vo1;
      }
      end1 = end0;
      end0 = seq;
      ++seg;
    }
    --seg;  // hand_over tags what is left with the last segment
    cp_async_wait<0>();
    if (ok) drain_all();
  } else if (some && warp == kMmaWarp) {
    // ----------------------------------- MMA -----------------------------------
    if (lane == 0) {
      constexpr uint32_t idS = idesc_fmt(BR, BK, FMT, false), idPV = idesc_fmt(BR, HD, FMT, true);
      bool ok = true;
      uint32_t base = 0, seg = 0, pc[2] = {0, 0};  // ring tiles before the segment; P tiles waited for
      auto take = [&](int at, unsigned code) {
        const uint32_t n = base + at;
        ok = ok && wait_abort(TMA ? &ready[n % NS] : &full[n % NS], (n / NS) & 1, p.err, code, abort_flag);
        if (ok) tc::fence_after_sync();
        return sRing + (n % NS) * C::kTile;
      };
      auto release = [&](int at) { tc::commit(&empty[(base + at) % NS]); };
      auto issue_s = [&](int u, const uint8_t* k) {
        const uint8_t* q = sQ + (PAIR ? u : seg & 1) * C::kTile;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_ss<FMT>(tmem + 256 * u, tc::desc_kmajor_sw128(q + (kk >> 2) * C::kAtom + (kk & 3) * 32),
                      tc::desc_kmajor_sw128(k + (kk >> 2) * C::kAtom + (kk & 3) * 32), idS, kk != 0);
        tc::commit(&s_full[u]);
      };
      auto issue_pv = [&](int u, const uint8_t* v, bool first) {
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          mma_ts<FMT>(tmem + 256 * u + 128, tmem + 256 * u + p_column(BIAS) + kk * 8,
                      tc::smem_desc(v + kk * 16 * 128, C::kAtom, 1024, tc::kSwizzle128B), idPV, !first || kk != 0);
      };
      auto wait_p = [&](int u) {
        ok = ok && wait_abort(&p_ready[u], pc[u] & 1, p.err, 0xB2400006u, abort_flag);
        ++pc[u];
        if (ok) tc::fence_after_sync();
      };
      while (ok && walk.next(p, tokens, sg)) {
        const int n = sg.n;
        const int units = PAIR && (2 * sg.rt + 1) * p.tpt < p.T ? 2 : 1;  // PAIR: row tiles of this item
        if constexpr (PAIR) {
          const uint8_t* k = take(0, 0xB2400004u);
          if (!ok) break;
          for (int u = 0; u < units; ++u) issue_s(u, k);
          release(0);
          for (int j = 0; j < n && ok; ++j) {
            const uint8_t* v = take(v_at(j, n), 0xB2400005u);
            const bool more = j + 1 < n;
            if (ok && more) k = take(k_at(j + 1), 0xB2400004u);
            for (int u = 0; u < units && ok; ++u) {
              wait_p(u);
              if (!ok) break;
              issue_pv(u, v, j == 0);
              if (!more) tc::commit(&o_done[u]);
              else issue_s(u, k);
            }
            if (!ok) break;
            release(v_at(j, n));
            if (more) release(k_at(j + 1));
          }
        } else {
          for (int j = 0; j < min(n, 2) && ok; ++j) {
            const uint8_t* k = take(k_at(j), 0xB2400004u);
            if (!ok) break;
            issue_s(j, k);
            release(k_at(j));
          }
          for (int j = 0; j < n && ok; ++j) {
            const int u = j & 1;
            const uint8_t* v = take(v_at(j, n), 0xB2400005u);
            if (ok) wait_p(u);
            if (!ok) break;
            issue_pv(u, v, j < 2);
            release(v_at(j, n));
            if (j + 2 >= n) {
              tc::commit(&o_done[u]);
            } else {
              const uint8_t* k = take(k_at(j + 2), 0xB2400004u);
              if (!ok) break;
              issue_s(u, k);
              release(k_at(j + 2));
            }
          }
        }
        base += 2 * n;
        ++seg;
      }
      if (!ok) {
        tc::commit(drain);
        mbar_wait(drain, 0, p.err, 0xB2400008u);
      }
    }
  } else if (some && warp >= 4) {
    // --------------------------------- softmax ---------------------------------
    const int u = (warp - 4) >> 2, qw = warp & 3, r = qw * 32 + lane;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const uint32_t tS = tmem + 256 * u + lane_off, tO = tmem + 128 + lane_off;  // tO: of unit 0
    Score score = make_score(p.softcap);
    uint32_t sc = 0, oc[2] = {0, 0}, seg = 0;  // S tiles / O accumulators waited for
    bool ok = true;
    while (walk.next(p, tokens, sg)) {
      const int rt = PAIR ? 2 * sg.rt + u : sg.rt;
      const int units = PAIR ? ((2 * sg.rt + 1) * p.tpt < p.T ? 2 : 1) : min(sg.n, 2);
      const int copy = r / rw, row = r - copy * rw;
      const int tt = row / p.rep, t = rt * p.tpt + tt, head = sg.hk * p.rep + row - tt * p.rep;
      const bool row_in = row < br && t < p.T, row_ok = row_in && t < sg.dl;
      // tokens of this warp; a warp without one leaves its P rows as they are
      // (their O is never read)
      const int w0 = qw * 32 & (rw - 1);
      const int t0 = rt * p.tpt + w0 / p.rep, t1 = min(rt * p.tpt + min((w0 + 31) / p.rep, p.tpt - 1), sg.dl - 1);
      const bool warp_ok = t0 < sg.dl && w0 < br, warp_in = t0 < p.T && w0 < br;
      const uint8_t* mask = p.mask ? p.mask + sg.b * p.mask_stride : nullptr;
      if constexpr (BIAS) score.slope0 = score.slope = row_in ? p.slopes[head] * attn::kLog2e : 0.f;
      // mask bits of the first 128 drafted tokens, read while the first keys are
      // still on their way (wider trees read theirs tile by tile)
      uint32_t drafted[4] = {0, 0, 0, 0};
      if (warp_ok && (sg.tile + sg.n) * BK > sg.ctx)
        draft_bits(drafted, mask, p.T, t, t0, t1, 0, min(sg.dl, 128));
      float m_used = -INFINITY, l = 0.f;
      bool first = true;
      const int step = PAIR ? 1 : 2;
      // at most 8 rows, each in a lane of its own in every warp (copies == 4): single
      // tokens with cap and bias in pages of 32 take 222 us this way, 278 the other
      const bool few = !PAIR && p.T * p.rep <= 8;
      // rows 8 to 23 of a copy's place in Q's tile are none
      uint8_t* room = sQ + (seg & 1) * C::kTile + (qw * 32 + 8 + 8 * u) * 128;
      for (int j = PAIR ? (u < units ? 0 : sg.n) : u; j < sg.n && ok; j += step) {
        ok = __all_sync(0xffffffffu, wait_abort(&s_full[u], sc & 1, p.err, 0xB2400009u, abort_flag));
        ++sc;
        if (!ok) break;
        tc::fence_after_sync();
        if (warp_ok) {
          const int kv0 = key_tile(j) * BK;
          uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
          if (kv0 + BK > sg.ctx) {
            visible_bits(vis, drafted, kv0 - sg.ctx);
            if (sg.dl > 128 && kv0 + BK > sg.ctx + 128) {
              uint32_t more[4];
              draft_bits(more, mask, p.T, t, t0, t1, kv0 - sg.ctx, sg.dl);
#pragma unroll
              for (int w = 0; w < 4; ++w) vis[w] |= more[w];
            }
          }
          // rows that are none see nothing: what stands in their place in Q's tile
          // must neither raise a maximum nor keep the warp from the short form of
          // the cap
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (!row_ok || (!PAIR && w * copies / 4 != copy)) vis[w] = 0;
          // SINGLE has no way of its own for whole tiles: it doubles the code of the
          // inner loop, whose instruction fetches then set its pace (single tokens
          // with cap and bias over 1 GB of cache: 360 us with it, 284 us without)
          const bool whole = PAIR && whole_tile(vis);
          // single tokens only: every visible key is at or before the row's own
          if constexpr (BIAS) score.dist = (float)(sg.ctx - kv0);
          if (few) softmax_few<HD, FMT, CAP, BIAS>(room, tS, tO + 256 * u, qw, word_of(vis, qw), score, !first, m_used, l);
          else softmax_tile<PAIR, HD, FMT, CAP, BIAS>(tS, tO + 256 * u, vis, whole, true, score, !first, m_used, l);
          tmem_st_wait();
        }
        first = false;
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[u]);
      }
      // ------------------------------ segment end ------------------------------
      // This thread writes row r: SINGLE, columns of half u from both units'
      // accumulators; PAIR, all columns of its own.
      if (few) {  // each row's sums to the thread that has it
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (lane >= 8) {
          m_used = -INFINITY;
          l = 0.f;
        }
      }
      float M = m_used, L = l, f0 = 1.f, f1 = 0.f;
      if constexpr (!PAIR) {
        s_ml[u * 128 + r] = make_float2(m_used, l);
        softmax_sync();
        for (int i = 0; i < 2 * copies; ++i) M = fmaxf(M, s_ml[(i & 1) * 128 + (i >> 1) * rw + row].x);
        const float ref = M == -INFINITY ? 0.f : M;
        L = f0 = 0.f;
        for (int i = 0; i < 2 * copies; ++i) {
          const float2 ml = s_ml[(i & 1) * 128 + (i >> 1) * rw + row];
          const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - ref);
          L = fmaf(ml.y, f, L);
          if (i >> 1 == copy) (i & 1 ? f1 : f0) = f;
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if ((PAIR && x != u) || x >= units) continue;
        ok = ok && __all_sync(0xffffffffu, wait_abort(&o_done[x], oc[x] & 1, p.err, 0xB240000Au, abort_flag));
        ++oc[x];
      }
      const bool whole = sg.n == sg.of;  // else a partial: before the run's first item border, or behind its last
      const bool bad = s_bad[seg & 1] == seg;
      const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
      float* part = p.ws + (2 * (int64_t)blockIdx.x + (sg.tile == 0 ? 1 : 0)) * (kRows * (HD + 2));
      // A drafted token's V that is infinite or NaN, for the rows that see it
      // (columns c .. c + N - 1)
      auto add_bad = [&](float* o, int c, int N) {
        const int j0 = max(sg.tile * BK - sg.ctx, 0), j1 = min((sg.tile + sg.n) * BK - sg.ctx, sg.dl);
        for (int j = j0; j < j1; ++j) {
          int64_t ko, vo;
          if (mask && !mask[(int64_t)t * p.T + j]) continue;
          if (!key_offset(p, sg.b, sg.hk, sg.ctx + j, key_page(p, sg.b, sg.ctx + j), ko, vo)) continue;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const uint16_t h = p.v[vo + c + e];
            if (not_finite16<FMT>(h)) o[e] += widen16<FMT>(h);
          }
        }
      };
      // Kinds of the 8 columns from c on in the context of this segment, of every n-th
      // key from the i-th on.
      auto context_kinds = [&](int c, int i, int n) {
        Kinds k = {0, 0, 0};
        const int end = min((sg.tile + sg.n) * BK, sg.ctx);
#pragma unroll 4
        for (int key = sg.tile * BK + i; key < end; key += n) {
          int64_t ko, vo;
          if (!key_offset(p, sg.b, sg.hk, key, key_page(p, sg.b, key), ko, vo)) continue;
          find_kinds<FMT>(*reinterpret_cast<const uint4*>(p.v + vo + c), k);
        }
        __syncwarp();
        return k;
      };
      auto drafted_bad = [&](int c) {  // what add_bad adds to one column
        const int j0 = max(sg.tile * BK - sg.ctx, 0), j1 = min((sg.tile + sg.n) * BK - sg.ctx, sg.dl);
        float x = 0.f;
        for (int j = j0; j < j1; ++j) {
          int64_t ko, vo;
          if (mask && !mask[(int64_t)t * p.T + j]) continue;
          if (!key_offset(p, sg.b, sg.hk, sg.ctx + j, key_page(p, sg.b, sg.ctx + j), ko, vo)) continue;
          if (not_finite16<FMT>(p.v[vo + c])) x += widen16<FMT>(p.v[vo + c]);
        }
        return x;
      };
      if (!PAIR && copies > 1) {
        // Copies: each warp stages its rows' sums over the units, CW columns at a
        // time, and the warpgroup adds the copies up on the way out.  A copy's weight
        // is 0 for the other copies' keys, which makes NaN of an infinity in their V:
        // where a sum is not finite, the columns of V that hold any in this segment's
        // context are looked up (all rows see the context), and such a column's sum is
        // the sum of those values, whatever their weights.  That reads V once more,
        // HD / 2 columns by each warpgroup, 32 or 64 keys at a time: 64 requests of up
        // to 8192 keys with an infinity in each, 32 / 8 heads of 128: 1.2 ms, not 0.25.
        if (!any_of_softmax(!ok)) {
          tc::fence_after_sync();
          constexpr int CW = HD == 128 ? 32 : 16, CPR = CW / 4;
          uint8_t* area = sQ + (seg & 1) * C::kTile + u * 128 * CW * 4;
          auto staged = [&](int rr, int ch) { return reinterpret_cast<float4*>(area + rr * CW * 4 + ((ch ^ (rr / (8 / CPR) & (CPR - 1))) << 4)); };
          if (!whole && u == 0 && copy == 0) {
            part[kRows * HD + row] = row_ok ? M : -INFINITY;
            part[kRows * HD + kRows + row] = row_ok ? L : 0.f;
          }
#pragma unroll 1
          for (int c = u * (HD / 2); c < (u + 1) * (HD / 2); c += CW) {
            float o[CW];
            float o1[CW];
            if constexpr (CW == 32) {
              tc::tmem_ld_32x32b_x32(tO + c, *reinterpret_cast<uint32_t(*)[32]>(o));
              if (units == 2) tc::tmem_ld_32x32b_x32(tO + 256 + c, *reinterpret_cast<uint32_t(*)[32]>(o1));
            } else {
              tmem_ld_32x32b_x16(tO + c, *reinterpret_cast<uint32_t(*)[16]>(o));
              if (units == 2) tmem_ld_32x32b_x16(tO + 256 + c, *reinterpret_cast<uint32_t(*)[16]>(o1));
            }
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < CW; ++e) {
              float x = f0 == 0.f ? 0.f : o[e] * f0;
              if (units == 2 && f1 != 0.f) x = fmaf(o1[e], f1, x);
              o[e] = x;
            }
            uint64_t zero2 = 0;  // NaN if one is not finite
#pragma unroll
            for (int e = 0; e < CW; e += 2) zero2 = fma_f2(f2_pack(o[e], o[e + 1]), 0, zero2);
            const float finite = f2_lo(zero2) + f2_hi(zero2);
            if (bad && row_ok && copy == 0) add_bad(o, c, CW);
            const float scale = whole ? inv : 1.f;
#pragma unroll
            for (int e = 0; e < CW; ++e) o[e] = row_ok && L != 0.f ? o[e] * scale : 0.f;
#pragma unroll
            for (int e = 0; e < CPR; ++e) *staged(r, e) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            // (a row whose weights add up to NaN is NaN anyway)
            if (__builtin_expect(any_of_warpgroup(u, row_ok && finite != 0.f && L == L), 0)) {
              constexpr int NL = CW / 8;  // threads a key
              const int part8 = (tid & 127) % NL;
              Kinds k = context_kinds(c + 8 * part8, (tid & 127) / NL, 128 / NL);
              uint32_t* found = reinterpret_cast<uint32_t*>(s_ml + u * 128);  // its sums are read: room for [4 warps][3]
              k.pos = __reduce_or_sync(0xffffffffu, k.pos << (8 * part8));
              k.neg = __reduce_or_sync(0xffffffffu, k.neg << (8 * part8));
              k.nan = __reduce_or_sync(0xffffffffu, k.nan << (8 * part8));
              if (lane == 0) {
                found[3 * qw] = k.pos;
                found[3 * qw + 1] = k.neg;
                found[3 * qw + 2] = k.nan;
              }
              warpgroup_sync(u);
              k.pos = found[0] | found[3] | found[6] | found[9];
              k.neg = found[1] | found[4] | found[7] | found[10];
              k.nan = found[2] | found[5] | found[8] | found[11];
              for (uint32_t left = k.any(); left; left &= left - 1) {
                const int e = __ffs(left) - 1;
                float x = 0.f;
                if (row_ok && copy == 0 && L != 0.f) {
                  x = k.sum(e);
                  if (bad) x += drafted_bad(c + e);
                  x *= scale;
                }
                reinterpret_cast<float*>(staged(r, e >> 2))[e & 3] = x;
              }
              warpgroup_sync(u);
            }
            for (int i = tid & 127; i < rw * CPR; i += 128) {
              const int rr = i / CPR, ch = i % CPR, t2 = rt * p.tpt + rr / p.rep;
              if (rr >= br || t2 >= p.T) continue;
              float4 a = *staged(rr, ch);
              for (int k = 1; k < copies; ++k) {
                const float4 b = *staged(rr + k * rw, ch);
                a.x += b.x;
                a.y += b.y;
                a.z += b.z;
                a.w += b.w;
              }
              if (whole) {
                uint16_t* to = p.o + sg.b * p.os[0] + (int64_t)t2 * p.os[1] + (int64_t)(sg.hk * p.rep + rr % p.rep) * p.os[2] + c + 4 * ch;
                *reinterpret_cast<uint2*>(to) = make_uint2(narrow2<FMT>(a.x, a.y), narrow2<FMT>(a.z, a.w));
              } else {
                *reinterpret_cast<float4*>(part + rr * HD + c + 4 * ch) = a;
              }
            }
            warpgroup_sync(u);
          }
        }
      } else if (ok && (!PAIR || u < units) && warp_in) {
        tc::fence_after_sync();
        constexpr int kCols = PAIR ? HD : HD / 2;
        const int c0 = PAIR ? 0 : u * kCols;
        // Rows leave through shared memory (Q's tile, which the segment no longer
        // needs): 32 rows of SB bytes a warp, so that a store instruction writes
        // whole 128-byte lines instead of 16 bytes of 32 rows.
        constexpr int SB = HD == 128 || PAIR ? 128 : 64, CPR = SB / 16;
        uint8_t* stage = sQ + (PAIR ? u : seg & 1) * C::kTile + (PAIR ? qw : 4 * u + qw) * 32 * SB;
        auto staged = [&](int rr, int ch) { return reinterpret_cast<uint4*>(stage + rr * SB + ((ch ^ (rr / (8 / CPR) & (CPR - 1))) << 4)); };
        uint8_t* dst = nullptr;  // of this lane's row
        if (whole) {
          if (row_in)
            dst = reinterpret_cast<uint8_t*>(p.o + sg.b * p.os[0] + (int64_t)t * p.os[1] + (int64_t)head * p.os[2]);
        } else {
          float* w = part;
          const int prow = PAIR ? u * BR + r : r;
          if (PAIR || u == 0) {
            w[kRows * HD + prow] = row_ok ? M : -INFINITY;
            w[kRows * HD + kRows + prow] = row_ok ? L : 0.f;
          }
          if (row_in) dst = reinterpret_cast<uint8_t*>(w + prow * HD);
        }
        auto flush = [&](int at) {  // SB bytes of every row, to byte `at` of it
          __syncwarp();
#pragma unroll
          for (int k = 0; k < CPR; ++k) {
            const int rr = k * (32 / CPR) + lane / CPR, ch = lane % CPR;
            uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), rr));
            if (to) *reinterpret_cast<uint4*>(to + at + ch * 16) = *staged(rr, ch);
          }
          __syncwarp();
        };
#pragma unroll 1
        for (int c = c0; c < c0 + kCols; c += 32) {
          float o[32];
          if constexpr (PAIR) {
            tc::tmem_ld_32x32b_x32(tO + 256 * u + c, *reinterpret_cast<uint32_t(*)[32]>(o));
            tc::tmem_ld_wait();
          } else {
            float o1[32];
            tc::tmem_ld_32x32b_x32(tO + c, *reinterpret_cast<uint32_t(*)[32]>(o));
            if (units == 2) tc::tmem_ld_32x32b_x32(tO + 256 + c, *reinterpret_cast<uint32_t(*)[32]>(o1));
            tc::tmem_ld_wait();
            // a factor of 0 belongs to a unit that saw nothing of this row: drop it
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              float x = f0 == 0.f ? 0.f : o[e] * f0;
              if (units == 2 && f1 != 0.f) x = fmaf(o1[e], f1, x);
              o[e] = x;
            }
          }
          if constexpr (FMT == kF16) {
            // A weight that rounds to 0 in fp16 (below 2^-25) makes NaN of an infinity,
            // as another copy's keys do above; one warp for its rows.
            float finite = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) finite = fmaf(o[e], 0.f, finite);
            if (__builtin_expect(__any_sync(0xffffffffu, row_ok && finite != 0.f && L == L), 0)) {
              Kinds k = context_kinds(c + 8 * (lane % 4), lane / 4, 8);
              k.pos = __reduce_or_sync(0xffffffffu, k.pos << (8 * (lane % 4)));
              k.neg = __reduce_or_sync(0xffffffffu, k.neg << (8 * (lane % 4)));
              k.nan = __reduce_or_sync(0xffffffffu, k.nan << (8 * (lane % 4)));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (k.any() >> e & 1) o[e] = k.sum(e);
            }
          }
          if (bad && row_ok) add_bad(o, c, 32);
          if (!row_ok || L == 0.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (whole) {  // 64 bytes of the row
            const int first = (c - c0) % (SB / 2) / 8;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *staged(lane, first + e) = make_uint4(narrow2<FMT>(o[8 * e] * inv, o[8 * e + 1] * inv),
                                                    narrow2<FMT>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                                    narrow2<FMT>(o[8 * e + 4] * inv, o[8 * e + 5] * inv),
                                                    narrow2<FMT>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
            if (first + 4 == CPR) flush((c + 32) * 2 - SB);
          } else {  // 128 bytes
#pragma unroll
            for (int h = 0; h < 8 / CPR; ++h) {
#pragma unroll
              for (int e = 0; e < CPR; ++e) {
                const float* x = o + h * (SB / 4) + 4 * e;
                *staged(lane, e) = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
              }
              flush(c * 4 + h * SB);
            }
          }
        }
      }
      ++seg;
      // both warpgroups have read the accumulators: the next segment may overwrite
      // them, and Q's tile, which the rows went through
      tc::fence_before_sync();
      if constexpr (TMA) tc::fence_proxy_async_smem();
      if (any_of_softmax(!ok)) break;
      if (lane == 0) mbar_arrive(&epi_done[(seg - 1) & 1]);
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// floor((a + b - 1) / b): 32-bit where it fits, since a 64-bit division costs
// about as much as a load from L2
__device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) {
  const int64_t n = a + b - 1;
  if (n >> 32 == 0) return (uint32_t)n / (uint32_t)b;
  return n / b;
}

// Joins the partials of the items that several CTAs shared:
// o = sum_c 2^{m_c - M} o_c / sum_c 2^{m_c - M} l_c.  One CTA per item and kJoin
// rows, four rows a warp, whose loads are in flight together.  Launched while
// the first kernel still runs (programmatic dependent launch): it finds its
// place in the schedule, then waits for that kernel's end.
constexpr int kJoin = 16;
template <int HD, int FMT, bool PAIR>
__global__ void __launch_bounds__(128) tree_join_kernel(const Params p, int64_t G) {
  constexpr int kRows = PAIR ? 2 * BR : BR;
  const int tokens = p.tpt * (PAIR ? 2 : 1);
  __shared__ int64_t s_w[4], s_before[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.y, rt = blockIdx.x % p.n_rt, hk = blockIdx.x / p.n_rt % p.Hkv;
  const int row0 = blockIdx.x / p.n_rt / p.Hkv * kJoin + warp * 4;
  int64_t W = 0, before = 0;
  for (int i = tid; i < p.B; i += 128) {
    const int64_t n = (int64_t)request(p, i, tokens).per_head * p.Hkv;
    W += n;
    if (i < b) before += n;
  }
  W = warp_sum(W);
  before = warp_sum(before);
  if (lane == 0) {
    s_w[warp] = W;
    s_before[warp] = before;
  }
  __syncthreads();
  W = s_w[0] + s_w[1] + s_w[2] + s_w[3];
  before = s_before[0] + s_before[1] + s_before[2] + s_before[3];
  const Req r = request(p, b, tokens);
  // before any way out, so that this kernel never ends before the first one
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (rt >= r.full) return;  // one tile: written by its CTA
  const int64_t g0 = before + (int64_t)hk * r.per_head + (int64_t)rt * (r.tiles + kItemCost) + kItemCost;
  const int64_t g1 = g0 + r.tiles;  // the item's tiles as units
  G = min(G, W);
  // CTA of unit g: the last one whose run starts at or before it
  const int ca = (int)ceil_div((g0 + 1) * G, W) - 1, cz = (int)ceil_div(g1 * G, W) - 1;
  if (ca == cz) return;  // a single segment: written by its CTA
  constexpr int V = HD / 32;  // columns a lane
  const int64_t stride = kRows * (HD + 2);
  float m[4], l[4], acc[4][V];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[i][e] = 0.f;
  }
  // (rows that are none of the item's read what lies there and are not stored)
  for (int c = ca; c <= cz; ++c) {
    const float* w = p.ws + (2 * (int64_t)c + (c == ca)) * stride;
    float mc[4], lc[4], x[4][V];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mc[i] = w[kRows * HD + row0 + i];
      lc[i] = w[kRows * HD + kRows + row0 + i];
      const float* o = w + (row0 + i) * HD + lane * V;
      if constexpr (V == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(o);
      else *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(o);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (lc[i] == 0.f) continue;  // saw nothing
      const float mn = fmaxf(m[i], mc[i]), ref = mn == -INFINITY ? 0.f : mn;
      const float fa = m[i] == -INFINITY ? 0.f : ex2(m[i] - ref), fb = ex2(mc[i] - ref);
      m[i] = mn;
      l[i] = l[i] * fa + lc[i] * fb;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[i][e] = acc[i][e] * fa + x[i][e] * fb;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int in = row0 + i, row = in % BR, t = (rt * (PAIR ? 2 : 1) + in / BR) * p.tpt + row / p.rep;
    if (row >= p.tpt * p.rep || t >= p.T) continue;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    uint16_t* o = p.o + b * p.os[0] + (int64_t)t * p.os[1] + (int64_t)(hk * p.rep + row % p.rep) * p.os[2] + lane * V;
    uint32_t h[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) h[e] = narrow2<FMT>(acc[i][2 * e] * inv, acc[i][2 * e + 1] * inv);
    if constexpr (V == 4) *reinterpret_cast<uint2*>(o) = make_uint2(h[0], h[1]);
    else *reinterpret_cast<uint32_t*>(o) = h[0];
  }
}

struct Maps {
  CUtensorMap q, k, v;
};

template <int HD, int FMT, bool PAIR, bool CAP, bool BIAS, bool TMA>
static void launch(const Maps& m, const Params& p, cudaStream_t st) {
  const int G = num_sms();
  set_max_smem((const void*)tree_kernel<HD, FMT, PAIR, CAP, BIAS, TMA>, Cfg<HD>::kSmem);
  tree_kernel<HD, FMT, PAIR, CAP, BIAS, TMA><<<G, kThreads, Cfg<HD>::kSmem, st>>>(m.q, m.k, m.v, p);
  const int rows = PAIR ? 2 * BR : (p.T < p.tpt ? p.T : p.tpt) * p.rep;
  const dim3 grid((unsigned)(p.n_rt * p.Hkv * ((rows + kJoin - 1) / kJoin)), p.B);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, tree_join_kernel<HD, FMT, PAIR>, p, (int64_t)G);
}

// Copies of the rows in a tile: as many as fit.  (64 requests of up to 8192 keys,
// four rows each, cap and bias, all by softmax_tile: 296 us with one copy, 283
// with four.)
inline int copies_of(int64_t rows) { return rows <= 32 ? 4 : rows <= 64 ? 2 : 1; }

// Launches by what the call has (BIAS: p.slopes, CAP: p.softcap).
void launch_tma(const Maps& m, const Params& p, int D, bool f16, bool pair, cudaStream_t st);
void launch_cp(const Maps& m, const Params& p, int D, bool f16, bool pair, cudaStream_t st);
template <bool TMA>
static void launch_form(const Maps& m, const Params& p, int D, bool f16, bool pair, cudaStream_t st) {
  const bool cap = p.softcap.log2 > 0.f, bias = p.slopes != nullptr;  // bias: single tokens, never pair
#define B2_TREE(HD, FMT)                                                                    \
  do {                                                                                      \
    if (pair && cap) launch<HD, FMT, true, true, false, TMA>(m, p, st);                     \
    else if (pair) launch<HD, FMT, true, false, false, TMA>(m, p, st);                      \
    else if (cap && bias) launch<HD, FMT, false, true, true, TMA>(m, p, st);                \
    else if (bias) launch<HD, FMT, false, false, true, TMA>(m, p, st);                      \
    else if (cap) launch<HD, FMT, false, true, false, TMA>(m, p, st);                       \
    else launch<HD, FMT, false, false, false, TMA>(m, p, st);                               \
  } while (0)
  if (D == 128 && f16) B2_TREE(128, fa::kF16);
  else if (D == 128) B2_TREE(128, fa::kBF16);
  else if (f16) B2_TREE(64, fa::kF16);
  else B2_TREE(64, fa::kBF16);
#undef B2_TREE
}
// launch_tma where tensor maps can describe the tensors, else launch_cp.
void launch_any(const Params& p, int64_t D, int64_t Hq, bool f16, bool pair, cudaStream_t st);
int launch_decode(const void* q, const void* k, const void* v, void* o, const int32_t* page_table,
                  const int32_t* seq_lens, void* workspace, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                  int64_t max_keys, int64_t page_size, int64_t max_pages, int64_t n_pages, const int64_t* k_strides,
                  const int64_t* v_strides, float scale, float softcap, const float* slopes, int dtype,
                  cudaStream_t st);

// Tensor maps of Q (dims d, head, token, request) and of K / V (contiguous:
// d, key, head, request; paged: d, head, token, page), boxes of one 128-byte
// swizzle row by the rows that the kernel's copies ask for.
bool make_maps(Maps& m, const Params& p, int64_t D, int64_t Hq, bool f16);
// Keys of a K / V box where the TMA form takes the cache, else 0.
int box_of(int64_t page_size, int64_t n_pages);
// Bytes of the workspace: two partials a CTA.
size_t workspace(int64_t T, int64_t rep, int64_t D);

}  // namespace tree
}  // namespace b2
