// tree_attention_tc.cuh — tree_attention.cuh's operator on tcgen05, for sequences whose
// rows (tokens x query heads of a key head) fill more of a 128-row MMA tile.
//
// A persistent CTA takes an equal share of all 128-key tiles of the call (TaShare): runs
// of tiles of consecutive segments (sequence, key head, QT x 128 rows).
//
//   warp 13      loader: page lookups, and TMA copies of K and V.  16-bit rows go straight
//                into the MMA's swizzled layout (boxes of 8 to 64 rows of one page); runs of
//                8-bit rows land in a ring of tiles, with their steps.
//   warps 0-3    8-bit rows (with warps 16-19): widen them to f16 in the MMA's layout.  16-bit
//                rows: zero what must not reach a product in a sequence's last tiles; or, where
//                the page size is no multiple of eight rows, load all rows themselves with
//                cp.async.
//   warps 4-11   softmax of unit 0 (4-7) and 1 (8-11), one row per thread (TMEM lane).
//                QT = 2: a unit is a tile of 128 rows and sees every key tile.  QT = 1: both
//                units share the rows and take alternate key tiles, joined at the end.
//   warp 12      MMA issuer (14, 15 are idle): O_t += P_t V of a unit's tile, then S_t = Q K^T
//                of its next one, while the other unit is in its softmax.
//
// Tensor memory: S_0 [0,128), S_1 [128,256), O_0 [256, 256+D), O_1 [256+D, 256+2D).  A
// softmax row walks its 128 scores twice, 64 at a time, and writes the weights P_t, two 16-bit
// values a column, over S_t, from where the second product reads them (its A operand);
// shared memory is left to K and V.  bf16 values need bf16 weights, whose eight bits would
// double the output's rounding: each 32 columns keep the weights' next eight bits in their
// second half, and a second product adds them.
// K and V are produced in the order in which the MMAs consume them.
//
// Measured (8 trees of 48 nodes over up to 16000 keys, 8 key heads of 128, 192 rows: 37 tiles a
// CTA): f16 115 us (3.4 TB/s), of a tile 2300 cycles softmax of a unit; e4m3 212 us at 1965 MHz,
// 11,200 cycles a tile, of which a unit's softmax takes 5400, for two steps a key (four widening
// warps instead of eight: 243 us).  2 trees of 16 nodes over 131000 keys, 4 key heads of 128,
// bf16, 46 tiles a CTA: 105 us after a pause, 116 in a loop that the power cap holds at 1640 MHz
// (3.9 TB/s; 4100 cycles a tile, of which scores, product and the product of the weights' low
// bits take 1536).  What the rest of a tile waits for has not been counted warp by warp.
// Registers: the 8-bit forms spill 44 to 84 bytes a thread at their 96, the 16-bit ones 4.
#pragma once
#include "tree_attention.cuh"

namespace ojx {

constexpr int TC_BN = 128;
constexpr int TC_PRODUCERS = 128;
// Threads and registers a thread: 16-bit caches 512 with 128 at launch (65,536), then
// 4 x 32 x (112 + 72) + 8 x 32 x 160 = 64,512; 8-bit caches 640 with 96 at launch (61,440), then
// 8 x 32 x 64 + 4 x 32 x 64 + 8 x 32 x 144 = 61,440.

template <int FMT, int D, int QT>
struct TcLayout {
  static constexpr bool QUANT = FMT >= TA_INT8;
  static constexpr int THREADS = QUANT ? 640 : 512;
  static constexpr int REGS_IN = QUANT ? 64 : 112, REGS_MMA = QUANT ? 64 : 72, REGS_SOFTMAX = QUANT ? 144 : 160;
  static constexpr int DB = D / 64;
  static constexpr int LEAD = QT == 1 ? 2 : 1;          // K tiles before the first V tile
  static constexpr int TILE = TC_BN * D * 2;            // a K or V tile as the MMA reads it
  static constexpr int BARS = 512;
  static constexpr int SLACK = 256;                     // to round the base up (it is aligned already, see the kernel)
  static constexpr int FIT = (227 * 1024 - BARS - SLACK - 2048 - QT * TILE) / TILE;  // tile buffers
  static constexpr int KST = QUANT ? 2 : D == 64 ? 4 : 3;
  static constexpr int VST = QUANT ? (D == 128 && QT == 2 ? 1 : 2) : D == 64 ? 4 : FIT - 3;
  static_assert(QUANT || KST + VST <= FIT, "shared memory");
  static constexpr int RAW = TC_BN * D;                 // a tile of 8-bit rows
  static constexpr int RAWS = !QUANT ? 0 : D == 64 ? 6 : 3;  // ring of them
  static constexpr int STEPS = !QUANT ? 0 : (QT == 1 ? 3 : 2) + KST;  // tiles whose steps are kept
  static constexpr int STEP_BYTES = 1568;
  static constexpr int RAWSTEP_RING = QUANT ? 4 : 0;
  static constexpr int OFF_K = QT * TILE;
  static constexpr int OFF_V = OFF_K + KST * TILE;
  static constexpr int OFF_RAW = OFF_V + VST * TILE;
  static constexpr int OFF_ROWS = OFF_RAW + RAWS * RAW;             // 4 x 128 row numbers (8 bits: and lengths)
  static constexpr int OFF_STEPS = OFF_ROWS + (QUANT ? 2 : 1) * 4 * 512;            // [STEPS][3][128] floats, [2][4] ints
  static constexpr int OFF_RAWSTEP = OFF_STEPS + STEPS * STEP_BYTES;
  static constexpr int OFF_BAR = OFF_RAWSTEP + RAWSTEP_RING * 1024;
  static constexpr int SMEM = OFF_BAR + BARS + SLACK;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void tc_sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
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

// The order in which a CTA's K and V tiles are produced, that of their use: within a part,
// V(i - lead) then K(i) for i = 0 .. n + lead - 1.
// `while (c.next(...))` visits them (one call site, so that the code exists once a role).
struct TcCursor {
  TaWalk walk;
  TaPart part;
  int i, lead;
  bool v;           // V or K
  uint32_t kc, vc;  // tiles of K and V before this one, over all parts
  __device__ __forceinline__ void begin(const TaWalk& w, int ahead) {
    walk = w;
    lead = ahead;
    part.n = 0;
    i = ahead;  // past a part without tiles
    v = true;
    kc = vc = 0xffffffffu;
    first = true;
  }
  bool first;
  __device__ __forceinline__ bool next(const TaParams& p, int per_seq) {
    if (first) {
      first = false;
      kc = vc = 0;
    } else if (v) {
      ++vc;
      v = false;
    } else {
      ++kc;
      v = true;
      ++i;
    }
    while (true) {
      if (i >= part.n + lead) {
        if (!walk.next(p, per_seq, TC_BN, part)) return false;
        i = 0;
        v = true;
      } else if (v && i < lead) {
        v = false;
      } else if (!v && i >= part.n) {
        v = true;
        ++i;
      } else {
        return true;
      }
    }
  }
  __device__ __forceinline__ uint32_t number() const { return v ? vc : kc; }
  __device__ __forceinline__ int tile() const { return part.t0 + (v ? i - lead : i); }
  __device__ __forceinline__ bool tail() const { return (tile() + 1) * TC_BN > part.ctx; }
  // Number (as K tile) of the V tile at the cursor: i - lead of the min(i, n) before it here.
  __device__ __forceinline__ uint32_t k_number() const { return kc - static_cast<uint32_t>(min(i, part.n) - (i - lead)); }
};

// MMAs and commits issued by the lane with `lead`, in a warp that runs together.  Shared-memory
// descriptors (128-byte swizzle): their constant parts for K and Q tiles and for V tiles; the
// address, in 16-byte units, joins the low word.
constexpr uint64_t tc_desc(uint32_t lbo, uint32_t sbo) {
  return (static_cast<uint64_t>(lbo >> 4) << 16) | (static_cast<uint64_t>(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint64_t SW128_K = tc_desc(16, 1024), SW128_V = tc_desc(8192, 1024);
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool add, bool lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(static_cast<uint32_t>(lead))
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool add, bool lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(static_cast<uint32_t>(lead))
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar, bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(static_cast<uint32_t>(lead))
      : "memory");
}

template <int FMT, int D, int QT>
__global__ void __launch_bounds__(TcLayout<FMT, D, QT>::THREADS, 1) tree_attention_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                          const __grid_constant__ CUtensorMap tmV,
                                                                          const TaParams p, uint64_t budget) {
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
  auto v_land = [&](int s) { return bar0 + 8u * (24 + s); };  // TMA of a tile to be cleaned
  auto raw_full = [&](int s) { return bar0 + 8u * (28 + s); };
  auto raw_empty = [&](int s) { return bar0 + 8u * (40 + s); };
  volatile int* s_abort = reinterpret_cast<volatile int*>(bars + 52);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 53);
  volatile int* s_odd = reinterpret_cast<volatile int*>(bars + 54);  // a hidden non-finite value was met
  TaShare* s_share = reinterpret_cast<TaShare*>(bars + 55);
  static_assert(55 * 8 + sizeof(TaShare) <= L::BARS && KST <= 4 && VST <= 4 && L::RAWS <= 12, "barrier area");
  const bool tma = !QUANT && p.box_rows > 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.tokens * p.group;
  const int per_seq = p.cache.kv_heads * p.row_tiles;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    mbar_init(done_bar, 1);
    for (int s = 0; s < KST; ++s) {
      mbar_init(k_full(s), tma ? 1 : QUANT ? 8 : 4);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(v_full(s), QUANT ? 8 : 4);
      mbar_init(v_empty(s), 1);
      mbar_init(v_land(s), 1);
    }
    for (int s = 0; s < L::RAWS; ++s) {
      mbar_init(raw_full(s), 33);
      mbar_init(raw_empty(s), 8);
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

  if (warp < 4 || warp >= 16) {
    // ── widening, cleaning, or loading by cp.async ─────────────────────────────────
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_IN));
    const int tid = warp < 4 ? threadIdx.x : threadIdx.x - 384;
    TaWalk walk;
    walk.begin(p, *s_share, TC_BN);
    TcCursor in;
    if constexpr (QUANT) {
      constexpr int CPR = D / 16, PER = TC_BN * CPR / 256;  // 16-byte pieces per row; per thread
      // Eight neighbouring threads take four pieces of each of two rows, from other halves of
      // the row: then neither their reads nor their two stores each meet a bank twice.
      const int col = D == 128 ? ((tid & 7) + ((tid >> 3) & 1) * 4) & 7 : tid % CPR;
      const int row0 = D == 128 ? (tid >> 4) * 2 + ((tid >> 2) & 1) : tid / CPR;
      uint32_t raw_n = 0;
      bool ok = true;
      in.begin(walk, LEAD);
      while (ok && in.next(p, per_seq)) {
        const bool v = in.v, tail = in.tail();
        const uint32_t n = in.number();
        const int left = in.part.ctx + in.part.drafts - in.tile() * TC_BN;  // rows that exist
        const int slot = raw_n % L::RAWS;
        ok = __all_sync(0xffffffffu, mbar_wait(raw_full(slot), (raw_n / L::RAWS) & 1u, budget, s_abort));
        if (!ok) break;
        ++raw_n;
        const uint4* raw = reinterpret_cast<const uint4*>(smem + L::OFF_RAW + slot * L::RAW) + row0 * CPR + col;
        uint4 w[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) w[i] = raw[i * 256];
        if (!v && warp < 4) {  // the row's steps, and the values' offset of the reference
          const float2 st = *reinterpret_cast<const float2*>(smem + L::OFF_RAWSTEP + (n & 3) * 1024 + tid * 8);
          float ks = st.x, vs = st.y;
          if (tail && !(fabsf(ks) < INFINITY && fabsf(vs) < INFINITY)) {
            ks = vs = 0.0f;  // as for the values: kept from rows that do not see the key
            *s_odd = 1;
          }
          float* d = reinterpret_cast<float*>(smem + L::OFF_STEPS + (n % L::STEPS) * L::STEP_BYTES) + tid;
          d[0] = ks == 0.0f ? 1.17549435e-38f : ks;  // (a row of zeros: its products are zero, and a hidden score stays -inf)
          d[128] = vs;
          d[256] = ta_step_log2(vs);
          // the largest and the smallest power of two among the rows' steps
          const int e = ta_step_exponent(vs);
          const int big = __reduce_max_sync(0xffffffffu, vs > 0.0f ? e : -1000);
          const int small = __reduce_min_sync(0xffffffffu, vs > 0.0f ? e : 1000);
          if (lane == 0) {
            int* range = reinterpret_cast<int*>(smem + L::OFF_STEPS + (n % L::STEPS) * L::STEP_BYTES + 1536);
            range[warp] = big;
            range[4 + warp] = small;
          }
        }
        if (tail) {
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (row0 + i * (256 / CPR) >= left) w[i] = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(raw_empty(slot));
        ok = __all_sync(0xffffffffu, mbar_wait(v ? v_empty(n % VST) : k_empty(n % KST), ((n / (v ? VST : KST)) & 1u) ^ 1u, budget, s_abort));
        if (!ok) break;
        const uint32_t to = v ? sV0 + (n % VST) * L::TILE : sK0 + (n % KST) * L::TILE;
        const int c = 2 * col;  // a piece becomes two 16-byte chunks of the widened row
        bool any = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int r = row0 + i * (256 / CPR);
          const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) ta_widen4<FMT>(x[e], y[2 * e], y[2 * e + 1]);
          if (FMT == TA_FP8 && tail) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (v) any |= tc_clean<false>(y[e]);
          }
          const uint32_t line = to + (v ? ((r >> 6) * L::DB + (c >> 3)) * 8192 + (r & 63) * 128 : (c >> 3) * 16384 + r * 128);
          tc_sts128(line + (((c & 7) ^ (r & 7)) << 4), y[0], y[1], y[2], y[3]);
          tc_sts128(line + ((((c + 1) & 7) ^ (r & 7)) << 4), y[4], y[5], y[6], y[7]);
        }
        if (any) *s_odd = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v ? v_full(n % VST) : k_full(n % KST));
      }
    } else if (tma) {
      // V tiles with drafts or the sequence's end: rows beyond the end hold whatever the page
      // does, and a hidden key's NaN or infinity would reach a row through 0 * value.  Both
      // are zeroed; the softmax warps give visible ones back.
      constexpr int CPR = D / 8;
      const int col = tid % CPR;
      uint32_t vn = 0, landed = 0;  // bit s: parity of stage s's next landing
      bool ok = true;
      TaPart part;
      while (ok && walk.next(p, per_seq, TC_BN, part)) {
        for (int j = max(0, part.ctx / TC_BN - part.t0); j < part.n && ok; ++j) {
          const uint32_t n = vn + j;
          // (a barrier of its own: these warps see only some of a stage's tiles)
          ok = __all_sync(0xffffffffu, mbar_wait(v_land(n % VST), (landed >> (n % VST)) & 1u, budget, s_abort));
          if (!ok) break;
          landed ^= 1u << (n % VST);
          const int left = part.ctx + part.drafts - (part.t0 + j) * TC_BN;
#pragma unroll 1
          for (int r = tid / CPR; r < TC_BN; r += 128 / CPR) {
            const uint32_t a = sV0 + (n % VST) * L::TILE + ((r >> 6) * L::DB + (col >> 3)) * 8192 + (r & 63) * 128 + (((col & 7) ^ (r & 7)) << 4);
            if (r >= left) {
              tc_sts128(a, 0, 0, 0, 0);
              continue;
            }
            uint4 x = ta_lds128(a);
            if (tc_clean<BF>(x.x) | tc_clean<BF>(x.y) | tc_clean<BF>(x.z) | tc_clean<BF>(x.w)) {
              tc_sts128(a, x.x, x.y, x.z, x.w);
              *s_odd = 1;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(v_full(n % VST));
        }
        vn += part.n;
      }
    } else {
      const uint8_t* kbase = static_cast<const uint8_t*>(p.cache.k);
      const uint8_t* vbase = static_cast<const uint8_t*>(p.cache.v);
      volatile int32_t* s_rows = reinterpret_cast<volatile int32_t*>(smem + L::OFF_ROWS);
      // Row numbers of the K tile at the cursor, for its copies and those of its V tile later.
      // The barrier also tells every producer whether one gave up, so that all stop together.
      bool fail = false;
      auto rows_of = [&]() {
        const int key = in.tile() * TC_BN + tid;
        int row = -1;
        if (key < in.part.ctx + in.part.drafts) {
          const int pg = key / p.cache.page_size;
          const int id = p.page_table[static_cast<int64_t>(in.part.b) * p.width + pg];
          if (id >= 0 && id < p.cache.num_pages)
            row = (id * p.cache.kv_heads + in.part.kvh) * p.cache.page_size + (key - pg * p.cache.page_size);
          else
            index_error();
        }
        s_rows[(in.kc & 3) * 128 + tid] = row;
        fail = named_bar_red_or(2, TC_PRODUCERS, fail);
      };
      constexpr int CPR = D / 8;                     // 16-byte chunks per row
      constexpr int COPIES = TC_BN * CPR / TC_PRODUCERS;
      constexpr int LAG = KST + VST - 1;             // groups in flight before the oldest is handed over
      const int col = tid % CPR;
      // groups committed and not yet handed over, oldest first: (is V, its number, in the tail)
      uint32_t q_item[LAG + 1] = {};
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
      in.begin(walk, LEAD);
      while (in.next(p, per_seq)) {
        const bool v = in.v;
        const uint32_t n = v ? in.vc : in.kc;
        if (!v) {
          rows_of();
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
        if (fail) continue;  // on to the next K tile's barrier
        const uint8_t* base = v ? vbase : kbase;
        const uint32_t tile = v ? in.k_number() : n;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
          const int r = tid / CPR + i * (TC_PRODUCERS / CPR);
          const int row = s_rows[(tile & 3) * 128 + r];
          ta_copy16(where(v, n, r), base + (row < 0 ? 0 : static_cast<int64_t>(row) * (D * 2) + col * 16), row >= 0);
        }
        ta_commit();
        const bool tail = in.tail();
#pragma unroll
        for (int i = 0; i <= LAG; ++i)
          if (i == pending) q_item[i] = (n << 2) | (tail ? 2u : 0u) | (v ? 1u : 0u);
        if (++pending > LAG) {
          ta_wait<LAG>();
          hand_over();
        }
      }
      ta_wait<0>();
      while (pending && !fail) hand_over();
    }
  } else if (warp >= 12) {
    // ── MMA issuer (warps 13-15 only give up registers) ────────────────────────
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_MMA));
    if (warp == 12) {
      // The whole warp runs the loop, with addresses from lane 0, and one lane issues: so the
      // descriptors stay in uniform registers.  (Issued from a branch of one lane, an MMA of
      // 32 cycles took a hundred.)
      constexpr uint32_t IDESC_S = make_idesc(MFMT, 0, 0, TC_BN, TC_BN);
      constexpr uint32_t IDESC_PV = make_idesc(MFMT, 0, 1, TC_BN, D);
      constexpr uint32_t HI_KV = static_cast<uint32_t>(SW128_K >> 32), LO_K = static_cast<uint32_t>(SW128_K);
      constexpr uint32_t HI_V = static_cast<uint32_t>(SW128_V >> 32), LO_V = static_cast<uint32_t>(SW128_V);
      const bool lead = lane == 0;
      auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
      const uint32_t uK = uniform(sK0 >> 4), uV = uniform(sV0 >> 4), uQ = uniform(sQ >> 4), uT = uniform(tmem);
      uint32_t kn = 0, pn[2] = {0, 0}, parts = 0;
      bool ok = true;
      TaWalk walk;
      walk.begin(p, *s_share, TC_BN);
      TaPart part;
      while (ok && walk.next(p, per_seq, TC_BN, part)) {
        const int n_tiles = static_cast<int>(uniform(part.n)), steps = QT * n_tiles;
        ok = __all_sync(0xffffffffu, mbar_wait(q_full, parts & 1u, budget, s_abort));
        ++parts;
        // (from -2: the first scores of both units; S_t of step i + 2 lies over P_t of step i,
        // and the MMAs run in order)
        for (int i = -2; i < steps && ok; ++i) {
          const int t = i & 1;
          if (i >= 0) {
            const uint32_t j = kn + (QT == 1 ? i : i >> 1), st = j % VST;
            if (QT == 1 || t == 0) ok = mbar_wait(v_full(st), (j / VST) & 1u, budget, s_abort);
            ok = ok && mbar_wait(p_full(t), pn[t] & 1u, budget, s_abort);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc_fence_after();
            const uint32_t b = LO_V | (uV + st * (L::TILE >> 4)), dO = uT + 2 * TC_BN + t * D, aP = uT + t * TC_BN;
#pragma unroll
            for (int ks = 0; ks < TC_BN / 16; ++ks) {
              const uint32_t at = b + (((ks >> 2) * (L::DB * 8192) + (ks & 3) * 2048) >> 4);
              tc_mma_ts(dO, aP + (ks >> 1) * 32 + (ks & 1) * 8, at, HI_V, IDESC_PV, i > 1 || ks > 0, lead);
              if constexpr (BF) tc_mma_ts(dO, aP + (ks >> 1) * 32 + (ks & 1) * 8 + 16, at, HI_V, IDESC_PV, true, lead);
            }
            ++pn[t];
            if (QT == 1 || t == 1) tc_commit(v_empty(st), lead);
            if (i + 2 >= steps) tc_commit(pv_done(t), lead);
          }
          if (i + 2 < steps) {
            const uint32_t j = kn + (QT == 1 ? i + 2 : (i + 2) >> 1), st = j % KST;
            if (QT == 1 || t == 0) ok = mbar_wait(k_full(st), (j / KST) & 1u, budget, s_abort);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc_fence_after();
            const uint32_t a = LO_K | (uQ + (QT == 1 ? 0 : t) * (L::TILE >> 4)), b = LO_K | (uK + st * (L::TILE >> 4));
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
              tc_mma_ss(uT + t * TC_BN, a + off, b + off, HI_KV, IDESC_S, ks > 0, lead);
            }
            tc_commit(s_full(t), lead);
            if (QT == 1 || t == 1) tc_commit(k_empty(st), lead);
          }
        }
        kn += n_tiles;
      }
      tc_commit(done_bar, lead);  // every MMA must complete before TMEM is released
      mbar_wait_drain(done_bar, 0, budget);
    } else if (warp == 13 && (QUANT || tma)) {
      // ── loader ─────────────────────────────────────────────────────────
      TcCursor c;
      {
        TaWalk walk;
        walk.begin(p, *s_share, TC_BN);
        c.begin(walk, LEAD);
      }
      bool ok = true;
      if constexpr (!QUANT) {
        // One box a lane: box_rows rows of one page x 64 columns.  Rows past the end start
        // outside the tensor and read as zeros.
        const int R = p.box_rows, ko = (lane / L::DB) * R, db = lane % L::DB;
        const bool on = lane < TC_BN / R * L::DB;
        const int rows_all = static_cast<int>(p.cache.num_pages) * p.cache.kv_heads * p.cache.page_size;
        uint32_t used = 0, parity = 0;  // bit s: K stage s, 8 + s: V stage s, 16 + s: its landings
        volatile int32_t* rows_at = reinterpret_cast<volatile int32_t*>(smem + L::OFF_ROWS) + lane;
        while (c.next(p, per_seq)) {
          const bool v0 = c.v, tail0 = c.tail();
          const uint32_t n0 = c.number();
          int row0;
          if (v0) {
            row0 = rows_at[(c.k_number() & 3) * 128];  // as found for the keys
          } else {
            const int key = c.tile() * TC_BN + ko;
            row0 = rows_all;
            if (on && key < c.part.ctx + c.part.drafts) {
              const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.cache.page_size;
              const int id = p.page_table[static_cast<int64_t>(c.part.b) * p.width + pg];
              if (id >= 0 && id < p.cache.num_pages)
                row0 = (id * p.cache.kv_heads + c.part.kvh) * p.cache.page_size + (key - pg * p.cache.page_size);
              else
                index_error();
            }
            rows_at[(n0 & 3) * 128] = row0;
          }
          const uint32_t st = n0 % (v0 ? VST : KST), ph = (n0 / (v0 ? VST : KST)) & 1u;
          ok = __all_sync(0xffffffffu, mbar_wait(v0 ? v_empty(st) : k_empty(st), ph ^ 1u, budget, s_abort));
          if (!ok) break;
          const uint32_t full = !v0 ? k_full(st) : tail0 ? v_land(st) : v_full(st);
          if (lane == 0) mbar_arrive_expect_tx(full, L::TILE);
          if (v0 && !tail0 && lane >= 1 && lane < 4) mbar_arrive(full);  // (v_full counts four, the cleaning warps)
          __syncwarp();
          if (on) {
            const uint32_t dst = v0 ? sV0 + st * L::TILE + ((ko >> 6) * L::DB + db) * 8192 + (ko & 63) * 128
                                    : sK0 + st * L::TILE + db * 16384 + ko * 128;
            tma_load_2d(dst, v0 ? &tmV : &tmK, full, db * 64, row0);
          }
          if (v0 && tail0) {  // phases of v_land count its own uses
            used = (used | 1u << (16 + st)) & ~(1u << (8 + st));  // (the stage's last load counts)
            parity ^= 1u << (16 + st);
          } else {
            used |= 1u << (v0 ? 8 + st : st);
            if (v0) used &= ~(1u << (16 + st));
            parity = (parity & ~(1u << (v0 ? 8 + st : st))) | (ph << (v0 ? 8 + st : st));
          }
        }
        __syncwarp();
        for (int s = 0; s < 4; ++s) {  // let every copy land before the CTA may exit
          if ((used >> s) & 1) mbar_wait_drain(k_full(s), (parity >> s) & 1, budget);
          if ((used >> (8 + s)) & 1) mbar_wait_drain(v_full(s), (parity >> (8 + s)) & 1, budget);
          if ((used >> (16 + s)) & 1) mbar_wait_drain(v_land(s), ((parity >> (16 + s)) & 1) ^ 1, budget);
        }
      } else {
        // A lane copies the runs of a page that start at its rows lane + 32 q of the tile.
        uint32_t raw_n = 0, used = 0, parity = 0;
        volatile int32_t* rows_at = reinterpret_cast<volatile int32_t*>(smem + L::OFF_ROWS) + lane;
        while (c.next(p, per_seq)) {
          const bool v0 = c.v;
          const uint32_t n0 = c.number(), ring = ((v0 ? c.k_number() : n0) & 3) * 256;
          int own[4], len[4];  // the key's row (-1: none), and the rows of the copy that starts there
          if (v0) {  // as found for the keys
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              own[q] = rows_at[ring + 64 * q];
              len[q] = rows_at[ring + 64 * q + 32];
            }
          } else {
            const int hi = c.part.ctx + c.part.drafts;
            int id[4], at[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int key = c.tile() * TC_BN + lane + 32 * q;
              id[q] = -1;
              at[q] = 0;
              if (key < hi) {
                const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.cache.page_size;
                at[q] = key - pg * p.cache.page_size;
                id[q] = p.page_table[static_cast<int64_t>(c.part.b) * p.width + pg];
                if (id[q] < 0) id[q] = INT32_MAX;
              }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int r = lane + 32 * q;
              own[q] = -1;
              len[q] = 0;
              if (id[q] >= p.cache.num_pages) {
                index_error();
              } else if (id[q] >= 0) {
                own[q] = (id[q] * p.cache.kv_heads + c.part.kvh) * p.cache.page_size + at[q];
                if (r == 0 || at[q] == 0) len[q] = min(min(p.cache.page_size - at[q], TC_BN - r), hi - c.tile() * TC_BN - r);
              }
              rows_at[ring + 64 * q] = own[q];
              rows_at[ring + 64 * q + 32] = len[q];
            }
          }
          const int slot = raw_n % L::RAWS;
          const uint32_t ph = (raw_n / L::RAWS) & 1u;
          ok = __all_sync(0xffffffffu, mbar_wait(raw_empty(slot), ph ^ 1u, budget, s_abort));
          if (!ok) break;
          const uint32_t full = raw_full(slot), dst = sbase + L::OFF_RAW + slot * L::RAW;
          const uint32_t bytes = __reduce_add_sync(0xffffffffu, (len[0] + len[1] + len[2] + len[3]) * D);
          if (lane == 0) mbar_arrive_expect_tx(full, bytes);
          __syncwarp();
          const uint8_t* base = static_cast<const uint8_t*>(v0 ? p.cache.v : p.cache.k);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (len[q]) bulk_load_g2s(dst + (lane + 32 * q) * D, base + static_cast<int64_t>(own[q]) * D, len[q] * D, full);
          if (!v0) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t d = sbase + L::OFF_RAWSTEP + (n0 & 3) * 1024 + (lane + 32 * q) * 8;
              ta_copy4(d, p.cache.k_scale + max(own[q], 0), own[q] >= 0);
              ta_copy4(d + 4, p.cache.v_scale + max(own[q], 0), own[q] >= 0);
            }
            tc_copies_arrive(full);
          } else {
            mbar_arrive(full);
          }
          used |= 1u << slot;
          parity = (parity & ~(1u << slot)) | (ph << slot);
          ++raw_n;
        }
        __syncwarp();
        for (int s = 0; s < L::RAWS; ++s)
          if ((used >> s) & 1) mbar_wait_drain(raw_full(s), (parity >> s) & 1, budget);
      }
    }
    __syncwarp();
  } else {
    // ── softmax ──────────────────────────────────────────────────────────
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_SOFTMAX));
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int lrow = quarter * 32 + lane;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    float2* s_ml = reinterpret_cast<float2*>(smem);  // [2][128], in Q's place between parts
    uint32_t steps_done = 0, tile_no = 0, ended = 0;  // this unit's steps, all key tiles, parts with a step, before the part
    bool ok = true;
    TaWalk walk;
    walk.begin(p, *s_share, TC_BN);
    TaPart part;
    while (walk.next(p, per_seq, TC_BN, part)) {
      const int kvh = part.kvh, rt = part.seg - kvh * p.row_tiles;
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
        const int k0 = (part.t0 + j) * TC_BN;
        if (k0 + TC_BN > part.ctx) {  // drafts, or the end: what the row does not see scores -inf
#pragma unroll 1
          for (int c = 0; c < TC_BN; c += 16) {
            const uint32_t see = ta_visible(p, part.b, token, k0 + c, part.ctx, hi);
            uint32_t w[16];
            tmem_ld16(trow + t * TC_BN + c, w);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = (see >> e) & 1 ? w[e] : 0xff800000u;
            tmem_st16(trow + t * TC_BN + c, w);
          }
          tmem_wait_st();
        }
        // Two passes over the scores in tensor memory, 64 columns an iteration: the loops stay
        // small, for what bounds a fully unrolled row is the fetching of its instructions.
        const ulonglong2* steps = reinterpret_cast<const ulonglong2*>(smem + L::OFF_STEPS + ((tile_no + j) % (L::STEPS ? L::STEPS : 1)) * L::STEP_BYTES);
        // Value steps of one tile seldom lie far apart: then the largest stands for all, and no
        // offset is read a key.
        float above = BF ? 0.0f : -TA_BIAS;
        bool narrow = true;
        if (QUANT) {
          const int4 big = *reinterpret_cast<const int4*>(steps + 96), small = *reinterpret_cast<const int4*>(steps + 97);
          const int hi_e = max(max(big.x, big.y), max(big.z, big.w)), lo_e = min(min(small.x, small.y), min(small.z, small.w));
          narrow = hi_e - lo_e <= TA_NEAR;
          above += static_cast<float>(hi_e > -1000 ? hi_e + 1 : TA_STEP_LOW);
        }
        const uint32_t tS = trow + t * TC_BN;
        const uint64_t rs2 = f2_pair(row_scale, row_scale);
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c0 = 0; c0 < TC_BN; c0 += 64) {
          uint32_t r[64];
#pragma unroll
          for (int c = 0; c < 64; c += 16) tmem_ld16(tS + c0 + c, *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
          tmem_wait_ld();
          if (narrow) {
#pragma unroll
            for (int c = 0; c < 64; c += 4) {
              float2 a = make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1]));
              float2 b = make_float2(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
              if (QUANT) {
                const ulonglong2 ks = steps[(c0 + c) / 4];
                a = f2_split(f2_mul(f2_pair(a.x, a.y), ks.x));
                b = f2_split(f2_mul(f2_pair(b.x, b.y), ks.y));
              }
              mx[(c >> 2) & 3] = fmaxf(fmaxf(mx[(c >> 2) & 3], fmaxf(a.x, a.y)), fmaxf(b.x, b.y));
            }
          } else {
#pragma unroll
            for (int c = 0; c < 64; c += 4) {  // (into the units of `top` below)
              const float4 ks = reinterpret_cast<const float4*>(steps)[(c0 + c) / 4], lv = reinterpret_cast<const float4*>(steps)[64 + (c0 + c) / 4];
              mx[0] = fmaxf(mx[0], fmaf(__uint_as_float(r[c]) * ks.x, row_scale, lv.x));
              mx[1] = fmaxf(mx[1], fmaf(__uint_as_float(r[c + 1]) * ks.y, row_scale, lv.y));
              mx[2] = fmaxf(mx[2], fmaf(__uint_as_float(r[c + 2]) * ks.z, row_scale, lv.z));
              mx[3] = fmaxf(mx[3], fmaf(__uint_as_float(r[c + 3]) * ks.w, row_scale, lv.w));
            }
          }
        }
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (narrow) top = fmaf(top, row_scale, above);  // (row_scale is positive: the largest stays the largest)
        else top -= TA_BIAS;
        const bool raise = valid && top > m_run + 8.0f;
        const float m_new = raise ? top : m_run;
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = raise ? ta_exp2(m_run - m_use) : 1.0f;
        const uint64_t neg2 = f2_pair(-m_use, -m_use);
        uint64_t sum2[2] = {0, 0};
        // (S_t in tensor memory means that the unit's last product is complete, O_t with it)
#pragma unroll 1
        for (int c0 = 0; c0 < TC_BN; c0 += 64) {
          uint32_t r[64];
#pragma unroll
          for (int c = 0; c < 64; c += 16) tmem_ld16(tS + c0 + c, *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
          tmem_wait_ld();
          // keys 32 k .. of the tile become columns 32 k .. 32 k + 15 (+ 16: their next bits)
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t hi_w[16], lo_w[BF ? 16 : 1];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              ulonglong2 ks = make_ulonglong2(0, 0), vs = ks;
              if (QUANT) {
                ks = steps[(c0 + c + e) / 4];
                vs = steps[32 + (c0 + c + e) / 4];
              }
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint64_t x = f2_pair(__uint_as_float(r[c + e + 2 * h]), __uint_as_float(r[c + e + 2 * h + 1]));
                if (QUANT) x = f2_mul(x, h ? ks.y : ks.x);
                const float2 a = f2_split(f2_fma(x, rs2, neg2));
                uint64_t w2 = f2_pair(ta_exp2(a.x), ta_exp2(a.y));
                sum2[h] = f2_add(sum2[h], w2);
                if (QUANT) w2 = f2_mul(w2, h ? vs.y : vs.x);
                const float2 w = f2_split(w2);
                const uint32_t pk = ta_pack(w.x, w.y, BF);
                hi_w[e / 2 + h] = pk;
                if (BF) lo_w[e / 2 + h] = ta_pack(w.x - __uint_as_float(pk << 16), w.y - __uint_as_float(pk & 0xffff0000u), true);
              }
            }
            tmem_st16(tS + c0 + c, hi_w);
            if constexpr (BF) tmem_st16(tS + c0 + c + 16, lo_w);
          }
        }
        float sum[4];
        {
          const float2 a = f2_split(sum2[0]), b = f2_split(sum2[1]);
          sum[0] = a.x, sum[1] = a.y, sum[2] = b.x, sum[3] = b.y;
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
            const int from = max(part.ctx / TC_BN, part.t0) * TC_BN, to = min(hi, (part.t0 + part.n) * TC_BN);
            for (int key = from; key < to; ++key) {
              if (!(ta_visible(p, part.b, token, key, part.ctx, hi) & 1)) continue;
              const int pg = key / p.cache.page_size;
              const int id = p.page_table[static_cast<int64_t>(part.b) * p.width + pg];
              if (id < 0 || id >= p.cache.num_pages) continue;
              const int64_t row = (static_cast<int64_t>(id) * p.cache.kv_heads + kvh) * p.cache.page_size + key % p.cache.page_size;
              const int64_t at = row * D + c;
              if (QUANT) {
                const float k0 = p.cache.k_scale[row] * 0.0f, v0 = p.cache.v_scale[row] * 0.0f;  // 0, or NaN
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[e] += k0 + v0;
              }
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

  grid_dep_launch_dependents();  // the join kernel may start; it waits for this grid's end
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ojx
