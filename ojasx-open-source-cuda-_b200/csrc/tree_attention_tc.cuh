// tree_attention_tc.cuh — tree_attention.cuh's operator on tcgen05, for sequences whose
// rows (tokens x query heads of a key head) fill more of a 128-row MMA tile.
//
// A persistent CTA takes an equal share of all 128-key tiles of the call (TaSplit): runs
// of tiles of consecutive segments (sequence, key head, QT x 128 rows).
//
//   warps 0-3    producers: page lookups, cp.async of K and V rows into the MMA's swizzled
//                layout; 8-bit rows land in a private ring first and are widened to f16.
//   warps 4-11   softmax of unit 0 (4-7) and 1 (8-11), one row per thread (TMEM lane).
//                QT = 2: a unit is a tile of 128 rows and sees every key tile.  QT = 1: both
//                units share the rows and take alternate key tiles, joined at the end.
//   warp 12      MMA issuer (13-15 are idle): O_t += P_t V of a unit's tile, then S_t = Q K^T
//                of its next one, while the other unit is in its softmax.
//
// Tensor memory: S_0 [0,128), S_1 [128,256), O_0 [256, 256+D), O_1 [256+D, 256+2D).  A
// softmax row holds its 128 scores in registers and writes the weights P_t, two 16-bit
// values a column, over S_t, from where the second product reads them (its A operand);
// shared memory is left to K and V.  bf16 values need bf16 weights, whose eight bits would
// double the output's rounding: columns 64-127 take the weights' next eight bits and a
// second product adds them.
// K and V are produced in the order in which the MMAs consume them.
#pragma once
#include "tree_attention.cuh"

namespace ojx {

constexpr int TC_BN = 128;
constexpr int TC_PRODUCERS = 128;
constexpr int TC_THREADS = 512;
// Registers a thread after the split: 128 at launch (65,536 / 512), then 4 x 32 x (80 + 56)
// + 8 x 32 x 184 = 64,512, within the launch's 65,536.

template <int FMT, int D, int QT>
struct TcLayout {
  static constexpr bool QUANT = FMT >= TA_INT8;
  static constexpr int DB = D / 64;
  static constexpr int LEAD = QT == 1 ? 2 : 1;          // K tiles before the first V tile
  static constexpr int TILE = TC_BN * D * 2;            // a K or V tile as the MMA reads it
  static constexpr int SLACK = 512;                     // to round the base up (it is aligned already, see the kernel)
  static constexpr int FIT = (227 * 1024 - 256 - SLACK - 2048 - QT * TILE) / TILE;  // tile buffers
  static constexpr int KST = QUANT ? 2 : D == 64 ? 4 : 3;
  static constexpr int VST = QUANT ? (D == 64 || QT == 1 ? 2 : 1) : D == 64 ? 4 : FIT - 3;
  static_assert(QUANT || KST + VST <= FIT, "shared memory");
  static constexpr int HALF = 64 * D;                   // half a tile of 8-bit rows
  static constexpr int HALVES = !QUANT ? 0 : D == 64 ? 12 : 6;    // ring of them
  static constexpr int STEPS = !QUANT ? 0 : (QT == 1 ? 3 : 2) + KST;  // tiles whose steps are kept
  static constexpr int RAWSTEP_RING = QUANT ? 4 : 0;
  static constexpr int OFF_K = QT * TILE;
  static constexpr int OFF_V = OFF_K + KST * TILE;
  static constexpr int OFF_RAW = OFF_V + VST * TILE;
  static constexpr int OFF_ROWS = OFF_RAW + HALVES * HALF;        // 4 x 128 row numbers
  static constexpr int OFF_STEPS = OFF_ROWS + 4 * 512;            // [STEPS][3][128] floats
  static constexpr int OFF_RAWSTEP = OFF_STEPS + STEPS * 1536;
  static constexpr int OFF_BAR = OFF_RAWSTEP + RAWSTEP_RING * 1024;
  static constexpr int SMEM = OFF_BAR + 256 + SLACK;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// ── the division of a call's key tiles over CTAs ──────────────────────────────────
// Sequence b has tiles(b) key tiles in each of its `per_seq` segments; tiles are counted
// sequence by sequence, segment by segment.  CTA c of G takes tiles [c U / G, (c+1) U / G).
// A segment's part that is not the whole segment goes to slot 0 of its CTA when it is the
// CTA's first, else to slot 1; the join kernel finds the parts from the same numbers.
struct TaLens {
  int ctx, drafts;
};
__device__ __forceinline__ TaLens ta_lens(const TaParams& p, int b, bool report) {
  int ctx = max(p.contexts[b], 0);
  int drafts = p.drafts ? min(max(p.drafts[b], 0), p.tokens) : p.tokens;
  const int64_t room = static_cast<int64_t>(p.width) * p.cache.page_size;
  if (static_cast<int64_t>(ctx) + drafts > room) {  // more keys than the page table holds
    if (report) index_error();
    ctx = static_cast<int>(min(static_cast<int64_t>(ctx), room));
    drafts = static_cast<int>(min(static_cast<int64_t>(drafts), room - ctx));
  }
  return {ctx, drafts};
}
__device__ __forceinline__ int ta_tiles(const TaParams& p, int b, int unit) {
  const TaLens l = ta_lens(p, b, false);
  return (l.ctx + l.drafts + unit - 1) / unit;
}

// Where a CTA's share begins: sequence, tiles before that sequence, first and last tile.
struct TaShare {
  int b;
  long long base, u, end;
};
// By one warp; the lanes take equal strips of sequences.
__device__ __forceinline__ TaShare ta_share_of(const TaParams& p, int per_seq, int unit, int cta, int ctas) {
  const int lane = threadIdx.x & 31;
  const int strip = (p.batch + 31) / 32;
  const int b0 = min(p.batch, lane * strip), b1 = min(p.batch, b0 + strip);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const TaLens l = ta_lens(p, b, cta == 0);
    mine += (l.ctx + l.drafts + unit - 1) / unit;
  }
  long long run = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  const long long total = __shfl_sync(0xffffffffu, run, 31) * per_seq;
  TaShare s;
  s.u = total * cta / ctas;
  s.end = total * (cta + 1) / ctas;
  s.b = 0;
  s.base = 0;
  const bool here = s.u < s.end && (run - mine) * per_seq <= s.u && s.u < run * per_seq;
  if (here) {
    long long base = (run - mine) * per_seq;
    int b = b0;
    for (; b < b1; ++b) {
      const long long n = static_cast<long long>(ta_tiles(p, b, unit)) * per_seq;
      if (s.u < base + n) break;
      base += n;
    }
    s.b = b;
    s.base = base;
  }
  const unsigned who = __ballot_sync(0xffffffffu, here);
  const int src = who ? __ffs(who) - 1 : 0;
  s.b = __shfl_sync(0xffffffffu, s.b, src);
  s.base = __shfl_sync(0xffffffffu, s.base, src);
  return s;
}

// One segment's part of a CTA's share.
struct TaPart {
  int b, seg, t0, n, tiles;  // sequence, segment in it, first tile, tiles here, tiles in all
  int ctx, drafts;
  bool first;                // first part of this CTA
};
struct TaWalk {
  TaShare s;
  int tiles, ctx, drafts;
  bool first;
  __device__ __forceinline__ void begin(const TaParams& p, const TaShare& share, int unit) {
    s = share;
    first = true;
    if (s.u < s.end) load(p, unit);
  }
  __device__ __forceinline__ void load(const TaParams& p, int unit) {
    const TaLens l = ta_lens(p, s.b, false);
    ctx = l.ctx;
    drafts = l.drafts;
    tiles = (ctx + drafts + unit - 1) / unit;
  }
  __device__ __forceinline__ bool next(const TaParams& p, int per_seq, int unit, TaPart& o) {
    if (s.u >= s.end) return false;
    while (s.u >= s.base + static_cast<long long>(tiles) * per_seq) {  // (ends: u < end <= all tiles)
      s.base += static_cast<long long>(tiles) * per_seq;
      ++s.b;
      load(p, unit);
    }
    const int at = static_cast<int>(s.u - s.base);
    o.b = s.b;
    o.seg = at / tiles;
    o.t0 = at - o.seg * tiles;
    o.tiles = tiles;
    o.n = static_cast<int>(min(static_cast<long long>(tiles - o.t0), s.end - s.u));
    o.ctx = ctx;
    o.drafts = drafts;
    o.first = first;
    first = false;
    s.u += o.n;
    return true;
  }
};

// Bits of keys k0 .. k0 + 31 that row `token` of sequence b sees (keys end at `hi`).
__device__ __forceinline__ uint32_t ta_visible(const TaParams& p, int b, int token, int k0, int ctx, int hi) {
  if (token < 0 || k0 >= hi) return 0;
  uint32_t bits = 0;
  const int d0 = k0 - ctx;
  if (d0 <= -32) {
    bits = 0xffffffffu;
  } else {
    const int from = max(d0, 0), lead = from - d0;  // first draft of the window, context keys before it
    uint32_t m;
    if (p.mask) {
      const int64_t* row = p.mask + b * p.mask_sb + static_cast<int64_t>(token) * p.words;
      const int w = from >> 6, sh = from & 63;
      uint64_t x = w < p.words ? static_cast<uint64_t>(row[w]) >> sh : 0;
      if (sh > 32 && w + 1 < p.words) x |= static_cast<uint64_t>(row[w + 1]) << (64 - sh);
      m = static_cast<uint32_t>(x);
    } else {
      const int n = token - from + 1;  // causal: drafts up to the row's own
      m = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
    }
    bits = lead == 0 ? m : (m << lead) | ((1u << lead) - 1u);
  }
  const int n = hi - k0;
  return n >= 32 ? bits : bits & ((1u << n) - 1u);
}

__device__ __forceinline__ void tc_sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float4 tc_lds4f(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
// Zeroes the non-finite 16-bit elements of a word; true if there were any.
template <bool BF>
__device__ __forceinline__ bool tc_clean(uint32_t& w) {
  constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
  bool any = false;
  if ((w & EXP) == EXP) w &= 0xffff0000u, any = true;
  if (((w >> 16) & EXP) == EXP) w &= 0x0000ffffu, any = true;
  return any;
}

template <int FMT, int D, int QT>
__global__ void __launch_bounds__(TC_THREADS, 1) tree_attention_tc_kernel(const TaParams p, uint64_t budget) {
  using L = TcLayout<FMT, D, QT>;
  constexpr bool QUANT = L::QUANT, BF = FMT == TA_BF16;
  constexpr int KST = L::KST, VST = L::VST, LEAD = L::LEAD;
  constexpr uint32_t MFMT = BF ? 1u : 0u;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  if (smem - smem_raw > L::SLACK) {  // (dynamic shared memory starts on a 1024-byte boundary)
    if (threadIdx.x == 0) atomicOr(&g_dev_error, OJX_DEVERR_TIMEOUT);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t sQ = sbase, sK0 = sbase + L::OFF_K, sV0 = sbase + L::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, done_bar = bar0 + 8;
  auto k_full = [&](int s) { return bar0 + 8u * (2 + s); };
  auto k_empty = [&](int s) { return bar0 + 8u * (6 + s); };
  auto v_full = [&](int s) { return bar0 + 8u * (10 + s); };
  auto v_empty = [&](int s) { return bar0 + 8u * (14 + s); };
  auto s_full = [&](int t) { return bar0 + 8u * (18 + t); };
  auto p_full = [&](int t) { return bar0 + 8u * (20 + t); };
  auto pv_done = [&](int t) { return bar0 + 8u * (22 + t); };
  volatile int* s_abort = reinterpret_cast<volatile int*>(bars + 24);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 25);
  volatile int* s_odd = reinterpret_cast<volatile int*>(bars + 26);  // a hidden non-finite value was met
  TaShare* s_share = reinterpret_cast<TaShare*>(bars + 27);
  static_assert(27 * 8 + sizeof(TaShare) <= 256 && KST <= 4 && VST <= 4, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.tokens * p.group;
  const int per_seq = p.cache.kv_heads * p.row_tiles;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    mbar_init(done_bar, 1);
    for (int s = 0; s < KST; ++s) {
      mbar_init(k_full(s), 4);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(v_full(s), 4);
      mbar_init(v_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t), 4);
      mbar_init(pv_done(t), 1);
    }
    *s_abort = 0;
    *s_odd = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(s_tmem), 512);
    tmem_relinquish();
  }
  if (warp == 0) {
    const TaShare s = ta_share_of(p, per_seq, TC_BN, blockIdx.x, gridDim.x);
    if (lane == 0) *s_share = s;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  TaWalk walk;
  walk.begin(p, *s_share, TC_BN);
  TaPart part;

  if (warp < 4) {
    // ── producers ────────────────────────────────────────────────────────
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    const int tid = threadIdx.x;
    const uint8_t* kbase = static_cast<const uint8_t*>(p.cache.k);
    const uint8_t* vbase = static_cast<const uint8_t*>(p.cache.v);
    volatile int32_t* s_rows = reinterpret_cast<volatile int32_t*>(smem + L::OFF_ROWS);
    // The sequence of copies: within a part, V(i - LEAD) then K(i) for i = 0 .. n + LEAD - 1.
    struct Cursor {
      TaWalk walk;
      TaPart part;
      int i;        // position in the part
      bool v, live;  // K or V next; anything left
      uint32_t kc, vc;  // tiles of K and V before this one, over all parts
    };
    auto settle = [&](Cursor& c) {  // move on to the next copy that exists
      while (c.live) {
        if (c.i >= c.part.n + LEAD) {
          c.live = c.walk.next(p, per_seq, TC_BN, c.part);
          c.i = 0;
          c.v = true;
        } else if (c.v && c.i < LEAD) {
          c.v = false;
        } else if (!c.v && c.i >= c.part.n) {
          c.v = true;
          ++c.i;
        } else {
          return;
        }
      }
    };
    auto advance = [&](Cursor& c) {
      if (c.v) {
        ++c.vc;
        c.v = false;
      } else {
        ++c.kc;
        c.v = true;
        ++c.i;
      }
      settle(c);
    };
    // Number (as K tile) of the V tile at the cursor: i - LEAD of the min(i, n) issued here.
    auto k_number = [&](const Cursor& c) { return c.kc - static_cast<uint32_t>(min(c.i, c.part.n) - (c.i - LEAD)); };
    // Row numbers of K tile `c`, for its copies and those of its V tile later.  The barrier
    // also tells every producer whether one of them gave up, so that all stop together.
    bool fail = false;
    auto rows_of = [&](const Cursor& c) {
      const int key = (c.part.t0 + c.i) * TC_BN + tid;
      int row = -1;
      if (key < c.part.ctx + c.part.drafts) {
        const int pg = key / p.cache.page_size;
        const int id = p.page_table[static_cast<int64_t>(c.part.b) * p.width + pg];
        if (id >= 0 && id < p.cache.num_pages)
          row = (id * p.cache.kv_heads + c.part.seg / p.row_tiles) * p.cache.page_size + (key - pg * p.cache.page_size);
        else
          index_error();
      }
      s_rows[(c.kc & 3) * 128 + tid] = row;
      fail = named_bar_red_or(2, TC_PRODUCERS, fail);
      return row;
    };
    Cursor in;
    in.walk = walk;
    in.i = 0;
    in.v = true;
    in.kc = in.vc = 0;
    in.live = in.walk.next(p, per_seq, TC_BN, in.part);
    settle(in);
    if constexpr (!QUANT) {
      constexpr int CPR = D / 8;                     // 16-byte chunks per row
      constexpr int COPIES = TC_BN * CPR / TC_PRODUCERS;
      constexpr int LAG = KST + VST - 1;             // groups in flight before the oldest is handed over
      const int col = tid % CPR;
      // groups committed and not yet handed over, oldest first: (is V, its number, in the tail)
      uint32_t q_item[LAG + 1];
      int pending = 0;
      auto where = [&](bool v, uint32_t n, int r) -> uint32_t {
        if (!v) return sK0 + (n % KST) * L::TILE + (col >> 3) * 16384 + r * 128 + (((col & 7) ^ (r & 7)) << 4);
        return sV0 + (n % VST) * L::TILE + ((r >> 6) * L::DB + (col >> 3)) * 8192 + (r & 63) * 128 + (((col & 7) ^ (r & 7)) << 4);
      };
      auto hand_over = [&]() {  // the oldest group has landed
        const uint32_t it = q_item[0];
        const bool v = it & 1, tail = it & 2;
        const uint32_t n = it >> 2;
        if (v && tail) {  // see tree_attention.cuh: hidden non-finite values must not reach a product
#pragma unroll 1
          for (int i = 0; i < COPIES; ++i) {
            const uint32_t a = where(true, n, tid / CPR + i * (TC_PRODUCERS / CPR));
            uint4 w = ta_lds128(a);
            const bool any = tc_clean<BF>(w.x) | tc_clean<BF>(w.y) | tc_clean<BF>(w.z) | tc_clean<BF>(w.w);
            if (any) {
              tc_sts128(a, w.x, w.y, w.z, w.w);
              *s_odd = 1;
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v ? v_full(n % VST) : k_full(n % KST));
#pragma unroll
        for (int i = 0; i < LAG; ++i) q_item[i] = q_item[i + 1];
        --pending;
      };
      while (in.live) {
        const bool v = in.v;
        const uint32_t n = v ? in.vc : in.kc;
        if (!v) {
          rows_of(in);
          if (fail) break;
        }
        const uint32_t bar = v ? v_empty(n % VST) : k_empty(n % KST);
        const uint32_t par = ((n / (v ? VST : KST)) & 1u) ^ 1u;
        if (!fail && !__all_sync(0xffffffffu, mbar_try_wait(bar, par))) {
          // the consumer is behind: nothing gained by holding finished copies back
          ta_wait<0>();
          while (pending) hand_over();
          fail = !__all_sync(0xffffffffu, mbar_wait(bar, par, budget, s_abort));
        }
        if (fail) {  // on to the next K tile's barrier
          advance(in);
          continue;
        }
        const uint8_t* base = v ? vbase : kbase;
        const uint32_t tile = v ? k_number(in) : n;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
          const int r = tid / CPR + i * (TC_PRODUCERS / CPR);
          const int row = s_rows[(tile & 3) * 128 + r];
          ta_copy16(where(v, n, r), base + (row < 0 ? 0 : static_cast<int64_t>(row) * (D * 2) + col * 16), row >= 0);
        }
        ta_commit();
        const int at = v ? in.i - LEAD : in.i;
        const bool tail = (in.part.t0 + at + 1) * TC_BN > in.part.ctx;
#pragma unroll
        for (int i = 0; i <= LAG; ++i)
          if (i == pending) q_item[i] = (n << 2) | (tail ? 2u : 0u) | (v ? 1u : 0u);
        if (++pending > LAG) {
          ta_wait<LAG>();
          hand_over();
        }
        advance(in);
      }
      ta_wait<0>();
      while (pending && !fail) hand_over();
    } else {
      // 8-bit rows: a thread copies 16-byte pieces into its own places of a ring of half
      // tiles, and later widens the pieces it copied (so no exchange is needed).
      constexpr int CPR = D / 16, PER = 64 * CPR / TC_PRODUCERS;  // pieces per row; per thread and half
      constexpr int RING = L::HALVES;
      const int col = tid % CPR, row0 = tid / CPR;
      const uint32_t raw = sbase + L::OFF_RAW, rawstep = sbase + L::OFF_RAWSTEP;
      Cursor out = in;
      int in_half = 0;
      uint32_t in_n = 0;
      auto issue = [&]() {
        if (in.live) {
          int row = 0;
          if (!in.v && in_half == 0) {
            row = rows_of(in);
            if (fail) in.live = false;
            const uint32_t d = rawstep + (in.kc % L::RAWSTEP_RING) * 1024 + tid * 8;
            ta_copy4(d, p.cache.k_scale + max(row, 0), row >= 0);
            ta_copy4(d + 4, p.cache.v_scale + max(row, 0), row >= 0);
          }
          const uint32_t tile = in.v ? k_number(in) : in.kc;
          const uint8_t* base = in.v ? vbase : kbase;
          const uint32_t slot = raw + (in_n % RING) * L::HALF;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int r = in_half * 64 + row0 + i * (TC_PRODUCERS / CPR);
            const int rr = s_rows[(tile & 3) * 128 + r];
            ta_copy16(slot + (i * TC_PRODUCERS + tid) * 16, base + (rr < 0 ? 0 : static_cast<int64_t>(rr) * D + col * 16), rr >= 0);
          }
          ++in_n;
          if (in_half == 0) {
            in_half = 1;
          } else {
            in_half = 0;
            advance(in);
          }
        }
        ta_commit();
      };
      for (int i = 0; i < RING; ++i) issue();
      uint32_t out_n = 0;
      while (out.live) {  // (after a failure: keeps step with the other producers' barriers)
        const bool v = out.v;
        const uint32_t n = v ? out.vc : out.kc;
        const int at = v ? out.i - LEAD : out.i;
        const bool tail = (out.part.t0 + at + 1) * TC_BN > out.part.ctx;
        if (!fail) fail = !__all_sync(0xffffffffu, mbar_wait(v ? v_empty(n % VST) : k_empty(n % KST), ((n / (v ? VST : KST)) & 1u) ^ 1u, budget, s_abort));
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          ta_wait<RING - 1>();
          if (fail) {
            ++out_n;
            issue();
            continue;
          }
          const uint32_t slot = raw + (out_n % RING) * L::HALF;
          uint4 w[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i) w[i] = ta_lds128(slot + (i * TC_PRODUCERS + tid) * 16);
          if (!v && half == 0) {  // the row's steps, and the values' offset of the reference
            const uint32_t d = rawstep + (n % L::RAWSTEP_RING) * 1024 + tid * 8;
            const float ks = ld_shared_f32(d), vs = ld_shared_f32(d + 4);
            const uint32_t to = sbase + L::OFF_STEPS + (n % L::STEPS) * 1536 + tid * 4;
            st_shared_f32(to, ks);
            st_shared_f32(to + 512, vs);
            st_shared_f32(to + 1024, fminf(fmaxf(__log2f(vs), -60.0f), 60.0f));
          }
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int r = half * 64 + row0 + i * (TC_PRODUCERS / CPR);
            const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[2 * e] = ta_widen<FMT>(x[e]);
              y[2 * e + 1] = ta_widen<FMT>(x[e] >> 16);
            }
            if (FMT == TA_FP8 && v && tail) {
              bool any = false;
#pragma unroll
              for (int e = 0; e < 8; ++e) any |= tc_clean<false>(y[e]);
              if (any) *s_odd = 1;
            }
            const int c = 2 * col;  // 16-byte chunk of the widened row
            const uint32_t line = v ? sV0 + (n % VST) * L::TILE + ((r >> 6) * L::DB + (c >> 3)) * 8192 + (r & 63) * 128 : sK0 + (n % KST) * L::TILE + (c >> 3) * 16384 + r * 128;
            tc_sts128(line + (((c & 7) ^ (r & 7)) << 4), y[0], y[1], y[2], y[3]);
            tc_sts128(line + ((((c + 1) & 7) ^ (r & 7)) << 4), y[4], y[5], y[6], y[7]);
          }
          ++out_n;
          issue();
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && !fail) mbar_arrive(v ? v_full(n % VST) : k_full(n % KST));
        advance(out);
      }
      ta_wait<0>();
    }
  } else if (warp >= 12) {
    // ── MMA issuer (warps 13-15 only give up registers) ────────────────────────
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 12 && lane == 0) {
      constexpr uint32_t IDESC_S = make_idesc(MFMT, 0, 0, TC_BN, TC_BN);
      constexpr uint32_t IDESC_PV = make_idesc(MFMT, 0, 1, TC_BN, D);
      uint32_t kn = 0, pn[2] = {0, 0}, parts = 0;
      bool ok = true;
      while (ok && walk.next(p, per_seq, TC_BN, part)) {
        const int steps = QT * part.n;
        ok = mbar_wait(q_full, parts & 1u, budget, s_abort);
        ++parts;
        auto issue_s = [&](int i) {
          const int t = i & 1;
          const uint32_t j = kn + (QT == 1 ? i : i >> 1);
          if ((QT == 1 || t == 0) && !mbar_wait(k_full(j % KST), (j / KST) & 1u, budget, s_abort)) return false;
          tc_fence_after();
          const uint32_t sK = sK0 + (j % KST) * L::TILE, sQt = sQ + (QT == 1 ? 0 : t) * L::TILE;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
            mma_f16(tmem + t * TC_BN, make_sw128_desc(sQt + off, 16, 1024), make_sw128_desc(sK + off, 16, 1024), IDESC_S,
                    ks > 0 ? 1u : 0u);
          }
          mma_commit(s_full(t));
          if (QT == 1 || t == 1) mma_commit(k_empty(j % KST));
          return true;
        };
        for (int i = 0; i < 2 && i < steps && ok; ++i) ok = issue_s(i);
        for (int i = 0; i < steps && ok; ++i) {
          const int t = i & 1;
          const uint32_t j = kn + (QT == 1 ? i : i >> 1);
          if ((QT == 1 || t == 0) && !(ok = mbar_wait(v_full(j % VST), (j / VST) & 1u, budget, s_abort))) break;
          if (!(ok = mbar_wait(p_full(t), pn[t] & 1u, budget, s_abort))) break;
          tc_fence_after();
          const uint32_t sV = sV0 + (j % VST) * L::TILE;
#pragma unroll
          for (int lo = 0; lo < (BF ? 2 : 1); ++lo)
#pragma unroll
            for (int ks = 0; ks < TC_BN / 16; ++ks) {
              const uint64_t bd = make_sw128_desc(sV + (ks >> 2) * (L::DB * 8192) + (ks & 3) * 2048, 8192, 1024);
              mma_f16_ts(tmem + 2 * TC_BN + t * D, tmem + t * TC_BN + lo * 64 + ks * 8, bd, IDESC_PV,
                         (i > 1 || ks > 0 || lo > 0) ? 1u : 0u);
            }
          ++pn[t];
          if (QT == 1 || t == 1) mma_commit(v_empty(j % VST));
          if (i + 2 < steps) ok = issue_s(i + 2);  // (over P_t: the MMAs run in order)
          else mma_commit(pv_done(t));
        }
        kn += part.n;
      }
      mma_commit(done_bar);  // every MMA must complete before TMEM is released
      mbar_wait_drain(done_bar, 0, budget);
    }
    __syncwarp();
  } else {
    // ── softmax ──────────────────────────────────────────────────────────
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int lrow = quarter * 32 + lane;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    float2* s_ml = reinterpret_cast<float2*>(smem);  // [2][128], in Q's place between parts
    uint32_t steps_done = 0, tile_no = 0, ended = 0;  // this unit's steps, all key tiles, parts with a step, before the part
    bool ok = true;
    while (walk.next(p, per_seq, TC_BN, part)) {
      const int kvh = part.seg / p.row_tiles, rt = part.seg % p.row_tiles;
      const int gr = rt * QT * TC_BN + (QT == 1 ? 0 : t * TC_BN) + lrow;
      const int itok = gr / p.group;
      const bool valid = gr < rows && itok < part.drafts;
      const int token = valid ? itok : -1;
      const bool busy = __any_sync(0xffffffffu, valid);  // a warp without rows only keeps step
      const int hi = part.ctx + part.drafts;

      // this row of Q (QT = 1: unit t writes half of it) into the swizzled tile
      float row_scale = p.scale_log2;
      {
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + part.b * p.q_sb + static_cast<int64_t>(valid ? itok : 0) * p.q_st +
                              static_cast<int64_t>(kvh * p.group + (valid ? gr % p.group : 0)) * p.q_sh;
        const bool wide = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && ((p.q_sb | p.q_st | p.q_sh) & 7) == 0;
        auto chunk = [&](int c) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (valid) {
            if (wide) {
              w = *reinterpret_cast<const uint4*>(src + c * 8);
            } else {
              uint32_t x[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = src[c * 8 + 2 * e] | (static_cast<uint32_t>(src[c * 8 + 2 * e + 1]) << 16);
              w = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
          return w;
        };
        auto as_f32 = [&](uint32_t h) {
          return p.dtype == OJX_BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
        };
        float up = 1.0f;
        if (QUANT && busy) {  // a power of two that brings the row into f16's range
          float amax = 0.0f;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = chunk(c);
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fmaxf(fabsf(as_f32(x[e] & 0xffffu)), fabsf(as_f32(x[e] >> 16))));
          }
          if (amax > 0.0f && amax < INFINITY) {
            const int ex = min(max(ilogbf(amax), -100), 100);
            up = exp2f(static_cast<float>(8 - ex));
            row_scale *= exp2f(static_cast<float>(ex - 8));
          }
        }
        constexpr int C0 = D / 8, PER = QT == 1 ? C0 / 2 : C0;
        if (busy) {
#pragma unroll 4
          for (int i = 0; i < PER; ++i) {
            const int c = (QT == 1 ? t * PER : 0) + i;
            uint4 w = chunk(c);
            if (QUANT) {
              uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = ta_pack(as_f32(x[e] & 0xffffu) * up, as_f32(x[e] >> 16) * up, false);
              w = make_uint4(x[0], x[1], x[2], x[3]);
            }
            tc_sts128(sQ + (QT == 1 ? 0 : t * L::TILE) + (c >> 3) * 16384 + lrow * 128 + (((c & 7) ^ (lrow & 7)) << 4), w.x, w.y, w.z, w.w);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }

      const int n_mine = QT == 1 ? (part.n - t + 1) / 2 : part.n;
      float m_run = -INFINITY, l_run = 0.0f;
      for (int k = 0; k < n_mine && ok; ++k) {
        const int j = QT == 1 ? 2 * k + t : k;
        const uint32_t step = steps_done + k;
        ok = __all_sync(0xffffffffu, mbar_wait(s_full(t), step & 1u, budget, s_abort));
        if (!ok) break;
        tc_fence_after();
        if (!busy) {
          if (lane == 0) mbar_arrive(p_full(t));
          continue;
        }
        uint32_t r[TC_BN];
#pragma unroll
        for (int c = 0; c < TC_BN; c += 16) tmem_ld16(trow + t * TC_BN + c, *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
        tmem_wait_ld();
        const int k0 = (part.t0 + j) * TC_BN;
        const bool all = k0 + TC_BN <= part.ctx;
        uint32_t see[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (!all) {
#pragma unroll
          for (int w = 0; w < 4; ++w) see[w] = ta_visible(p, part.b, token, k0 + 32 * w, part.ctx, hi);
        }
        const uint32_t steps = sbase + L::OFF_STEPS + ((tile_no + j) % (L::STEPS ? L::STEPS : 1)) * 1536;
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < TC_BN; c += 4) {
          float4 ks = make_float4(1, 1, 1, 1), lv = make_float4(0, 0, 0, 0);
          if (QUANT) {
            ks = tc_lds4f(steps + c * 4);
            lv = tc_lds4f(steps + 1024 + c * 4);
          }
          const float kk[4] = {ks.x, ks.y, ks.z, ks.w}, ll[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = __uint_as_float(r[c + e]);
            if (QUANT) {
              x *= kk[e];
              r[c + e] = __float_as_uint(x);
            }
            const float y = QUANT ? fmaf(x, row_scale, ll[e]) : x;
            if (all) mx[e] = fmaxf(mx[e], y);
            else if ((see[(c + e) >> 5] >> ((c + e) & 31)) & 1) mx[e] = fmaxf(mx[e], y);
          }
        }
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (!QUANT) top *= row_scale;  // positive: the largest stays the largest
        const bool raise = valid && top > m_run + 8.0f;
        const float m_new = raise ? top : m_run;
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = raise ? ta_exp2(m_run - m_use) : 1.0f;
        float sum[4] = {0, 0, 0, 0};
        // (S_t in tensor memory means that the unit's last product is complete, O_t with it)
#pragma unroll
        for (int c = 0; c < TC_BN / 8; ++c) {
          float vs[8];
          if (QUANT) {
            const float4 a = tc_lds4f(steps + 512 + c * 32), b4 = tc_lds4f(steps + 512 + c * 32 + 16);
            vs[0] = a.x, vs[1] = a.y, vs[2] = a.z, vs[3] = a.w, vs[4] = b4.x, vs[5] = b4.y, vs[6] = b4.z, vs[7] = b4.w;
          }
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const int kk = 8 * c + i;
            float e0 = ta_exp2(fmaf(__uint_as_float(r[kk]), row_scale, -m_use));
            float e1 = ta_exp2(fmaf(__uint_as_float(r[kk + 1]), row_scale, -m_use));
            if (!all) {
              e0 = (see[kk >> 5] >> (kk & 31)) & 1 ? e0 : 0.0f;
              e1 = (see[kk >> 5] >> ((kk + 1) & 31)) & 1 ? e1 : 0.0f;
            }
            sum[(kk >> 1) & 3] += e0 + e1;
            if (QUANT) {
              // (hidden: 0, whatever the step)
              e0 = !all && !((see[kk >> 5] >> (kk & 31)) & 1) ? 0.0f : e0 * vs[i];
              e1 = !all && !((see[kk >> 5] >> ((kk + 1) & 31)) & 1) ? 0.0f : e1 * vs[i + 1];
            }
            // pairs replace the scores in place: r[k] the weights, r[k + 1] their next bits
            const uint32_t w = ta_pack(e0, e1, BF);
            r[kk] = w;
            if (BF) r[kk + 1] = ta_pack(e0 - __uint_as_float(w << 16), e1 - __uint_as_float(w & 0xffff0000u), true);
          }
          if (c % 4 == 3) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = r[8 * (c - 3) + 2 * i];
            tmem_st16(trow + t * TC_BN + (c - 3) * 4, pk);
            if (BF) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = r[8 * (c - 3) + 2 * i + 1];
              tmem_st16(trow + t * TC_BN + 64 + (c - 3) * 4, pk);
            }
          }
        }
        l_run = l_run * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        m_run = m_new;
        if (k > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(trow + 2 * TC_BN + t * D + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(trow + 2 * TC_BN + t * D + c, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(t));
      }
      steps_done += n_mine;
      tile_no += part.n;
      if (ok && n_mine > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(pv_done(t), ended & 1u, budget, s_abort));
        tc_fence_after();
      }
      ended += n_mine > 0;
      if (!valid) m_run = -INFINITY, l_run = 0.0f;
      // ── the part's result (the barriers are taken on every path) ─────────────────
      float f[2] = {t == 0 ? 1.0f : 0.0f, t == 1 ? 1.0f : 0.0f};
      float top = m_run, l = l_run;
      if (QT == 1) {
        tc_fence_before();
        named_bar_sync(1, 256);  // both units' products are done: Q is free
        s_ml[t * TC_BN + lrow] = make_float2(m_run, l_run);
        named_bar_sync(1, 256);
        tc_fence_after();
        const float2 a = s_ml[lrow], c = s_ml[TC_BN + lrow];
        top = fmaxf(a.x, c.x);
        f[0] = ta_share(a.x, a.y, top);
        f[1] = ta_share(c.x, c.y, top);
        l = 0.0f;
        if (f[0] != 0.0f) l += f[0] * a.y;
        if (f[1] != 0.0f) l += f[1] * c.y;
      } else if (n_mine == 0) {
        f[t] = 0.0f;
      }
      const bool whole = part.n == part.tiles;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (part.first ? 0 : 1)) * (QT * TC_BN) + (QT == 1 ? 0 : t * TC_BN) + lrow;
      if (ok && busy) {
        const int c0 = QT == 1 ? t * (D / 2) : 0, c1 = QT == 1 ? c0 + D / 2 : D;
        const bool odd = *s_odd != 0;
#pragma unroll 1
        for (int c = c0; c < c1; c += 16) {
          float acc[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (QT == 2 && u != t) continue;
            uint32_t o[16];
            tmem_ld16(trow + 2 * TC_BN + u * D + c, o);
            tmem_wait_ld();
            if (f[u] != 0.0f) {
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[i] += f[u] * __uint_as_float(o[i]);
            }
          }
          if (odd && valid) {  // give the non-finite values to the rows that see them
            const int from = max(part.ctx, part.t0 * TC_BN), to = min(hi, (part.t0 + part.n) * TC_BN);
            for (int key = from; key < to; ++key) {
              if (!(ta_visible(p, part.b, token, key, part.ctx, hi) & 1)) continue;
              const int pg = key / p.cache.page_size;
              const int id = p.page_table[static_cast<int64_t>(part.b) * p.width + pg];
              if (id < 0 || id >= p.cache.num_pages) continue;
              const int64_t at = ((static_cast<int64_t>(id) * p.cache.kv_heads + kvh) * p.cache.page_size + key % p.cache.page_size) * D + c;
              for (int i = 0; i < 16; ++i) {
                float v;
                if (QUANT) v = dequantise_one(static_cast<const uint8_t*>(p.cache.v)[at + i], 1.0f, p.cache.format);
                else if (BF) v = __bfloat162float(static_cast<const __nv_bfloat16*>(p.cache.v)[at + i]);
                else v = __half2float(static_cast<const __half*>(p.cache.v)[at + i]);
                if (!(fabsf(v) < INFINITY)) {
#pragma unroll
                  for (int e = 0; e < 16; ++e)
                    if (e == i) acc[e] += v;
                }
              }
            }
          }
          if (gr < rows) {
            if (whole) {
              const int64_t at = ((static_cast<int64_t>(part.b) * p.tokens + itok) * p.q_heads + kvh * p.group + gr % p.group) * D + c;
              uint32_t pk[8];
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                pk[i / 2] = ta_pack(l == 0.0f ? 0.0f : acc[i] * inv, l == 0.0f ? 0.0f : acc[i + 1] * inv, p.dtype == OJX_BF16);
              uint4* d4 = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at);
              d4[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
              d4[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            } else {
              float4* d4 = reinterpret_cast<float4*>(p.part_o + slot * D + c);
#pragma unroll
              for (int i = 0; i < 4; ++i) d4[i] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
            }
          }
        }
        if (!whole && gr < rows && (QT == 2 || t == 0)) p.part_ml[slot] = make_float2(top, l);
      } else if (ok && whole && gr < rows && (QT == 2 || t == 0)) {
        // (a warp whose rows are all beyond the sequence's drafts)
        uint4* d4 = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) +
                                             ((static_cast<int64_t>(part.b) * p.tokens + itok) * p.q_heads + kvh * p.group + gr % p.group) * D);
        for (int c = 0; c < D / 8; ++c) d4[c] = make_uint4(0, 0, 0, 0);
      } else if (ok && !whole && gr < rows && (QT == 2 || t == 0)) {
        p.part_ml[slot] = make_float2(-INFINITY, 0.0f);
      }
      if (QT == 1) {
        tc_fence_before();
        named_bar_sync(1, 256);  // Q, s_ml and O are read: the next part may write them
        tc_fence_after();
      } else {
        tc_fence_before();
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of segments that more than one CTA took, and writes the zeros of
// sequences without keys.  One warp per row.
template <int D>
__global__ void __launch_bounds__(128) tree_attention_parts_kernel(const TaParams p, int tile_rows, int unit, int ctas) {
  const int lane = threadIdx.x & 31;
  const int rows = p.tokens * p.group;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= static_cast<int64_t>(p.batch) * p.cache.kv_heads * rows) return;
  const int r = static_cast<int>(w % rows);
  const int64_t bh = w / rows;
  const int b = static_cast<int>(bh / p.cache.kv_heads), kvh = static_cast<int>(bh % p.cache.kv_heads);
  const int per_seq = p.cache.kv_heads * p.row_tiles;
  long long before = 0, total = 0;
  for (int i = lane; i < p.batch; i += 32) {
    const int n = ta_tiles(p, i, unit);
    total += n;
    if (i < b) before += n;
  }
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  const int tiles = ta_tiles(p, b, unit);
  const int64_t at = ((static_cast<int64_t>(b) * p.tokens + r / p.group) * p.q_heads + kvh * p.group + r % p.group) * D;
  if (tiles == 0) {
    for (int i = 0; i < D / 32; ++i) store_as(p.out, at + lane + 32 * i, p.dtype, 0.0f);
    return;
  }
  total *= per_seq;
  const long long u0 = before * per_seq + static_cast<long long>(kvh * p.row_tiles + r / tile_rows) * tiles;
  auto owner = [&](long long u) { return static_cast<int>(((u + 1) * ctas - 1) / total); };
  const int c0 = owner(u0), c1 = owner(u0 + tiles - 1);
  if (c0 == c1) return;  // written by its CTA
  auto slot_of = [&](int c) {
    const int which = c > c0 || total * c / ctas == u0 ? 0 : 1;
    return (static_cast<int64_t>(c) * 2 + which) * tile_rows + r % tile_rows;
  };
  float top = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32)
    if (total * c / ctas < total * (c + 1) / ctas) top = fmaxf(top, p.part_ml[slot_of(c)].x);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float acc[D / 32], l = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
  for (int c = c0; c <= c1; ++c) {
    if (total * c / ctas >= total * (c + 1) / ctas) continue;  // a CTA without tiles
    const int64_t slot = slot_of(c);
    const float2 ml = p.part_ml[slot];
    const float f = ta_share(ml.x, ml.y, top);
    if (f != 0.0f) {
      l += f * ml.y;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] += f * p.part_o[slot * D + lane + 32 * i];
    }
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_as(p.out, at + lane + 32 * i, p.dtype, l == 0.0f ? 0.0f : acc[i] / l);
}

}  // namespace ojx
