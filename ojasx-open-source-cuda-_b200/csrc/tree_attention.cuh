// tree_attention.cuh — attention of a sequence's newest tokens over its paged cache: one
// token (decoding), a chunk, or a tree of drafts.
//
// Row (token i, query head h) of sequence b sees keys 0 .. context-1 and those drafts
// j < draft_len whose bit is set in mask[b][i] (no mask: j <= i); the drafts' keys lie at
// context + j.  out = sum_j softmax_j(scale q.k_j) v_j in one pass over the keys with a
// running reference and sum (fp32); a row that sees nothing gives zeros.
//
// A quantised key is an 8-bit vector times a step, so the products run on the stored
// values, which are exact in f16, and the step multiplies the score: s_j = step_kj * (q.k8_j).
// For the values the step joins the weight: sum_j (p_j step_vj) v8_j.  A row measures its
// weights against the largest s_j + log2(step_vj) instead of the largest s_j, so they use
// f16's range whatever the steps are (see TA_BIAS).  A bf16 query row is brought into f16's
// range by a power of two, which the score's factor takes back.
//
// Up to 16 rows a key head, this file: each key and value is read once, so HBM bounds 16-bit
// caches (64 sequences of up to 8191 keys, 8 key heads of 128, 4 rows: 223 us, 6.5 TB/s) and
// instructions bound 8-bit ones (int8 174 us, e4m3 193 us, 4.2 and 3.9 TB/s): widening, the
// products with half-empty fragments, and the softmax are about 1060 instructions a warp and
// block of 32 keys; half of the issue slots stay empty (fixed latencies).  With up to 8 rows of
// 128 the 8-bit forms spill (int8 56, e4m3 112 bytes a thread at 168 registers, which twelve
// warps leave).  Short calls are a chain of latencies (701 keys: 6.8 us).
#pragma once
#include "qk_cache.cuh"

namespace ojx {

struct TaParams {
  ojx_kv_cache cache;
  const void* q;
  void* out;
  int64_t q_sb, q_st, q_sh;
  int dtype, batch, tokens, q_heads, group;
  const int32_t* page_table;
  int width;
  const int32_t* contexts;
  const int32_t* drafts;
  const int64_t* mask;
  int64_t mask_sb;
  int words;
  float scale_log2;
  int row_tiles;
  int page_shift;  // log2 of the page size, or -1
  int box_rows;    // rows of a TMA box (16-bit caches on tcgen05), 0: no TMA
  float* part_o;    // [CTA][2][rows][D], unnormalised: the parts of segments that CTAs share
  float2* part_ml;  // [CTA][2][rows]: reference, sum
};

constexpr int TA_F16 = 0, TA_BF16 = 1, TA_INT8 = 2, TA_FP8 = 3;

// Weights enter the second product in f16 (over bf16 values: as two bf16 numbers): 11 bits,
// which is what the output's own rounding to f16 keeps; the sum of the weights stays in
// fp32.  (With a second product for their next bits, f16 queries over e4m3 were off by 2.1e-4
// of the output's norm instead of 2.9e-4, bf16 queries over int8 by 1.7e-3 either way; eight
// trees of 48 nodes took 267 us instead of 231, a decoding batch of 64 took 204 instead of
// 183 over int8, 240 instead of 202 over e4m3.)  A row's largest weight (times its value's step) lies near 2^7 when its reference is
// set and below 2^15 until the reference moves, so weights keep their 11 bits down to 2^-21
// of the largest and contribute down to 2^-31 of it: a long context whose keys share what
// one large score leaves is not lost.  (With the largest at one, and steps 2^8 apart taken
// as the largest of them, 65536 keys of 2^-16 of the largest weight each added nothing.)
constexpr float TA_BIAS = 7.0f;
// Value steps whose powers of two differ by no more than this are taken as the largest of
// their block, which costs that many of the bits above.  (Where all blocks' steps lie further
// apart, eight e4m3 trees of 48 nodes take 246 us instead of 231, an int8 decoding batch of 64
// takes 192 instead of 185.)
constexpr int TA_NEAR = 2;
// log2 of the value steps that weights are measured in.  Above, no product passes f16's range
// up to the largest float there is (2^121 a step); the weights' own sum keeps 2^-11 of the
// largest weight at 2^121, 2^-32 at 2^100.  Below, a sum of 2^17 weights stays in fp32's range;
// smaller steps lose the weights' bits one by one.
constexpr int TA_STEP_LOW = -90, TA_STEP_HIGH = 122;
__device__ __forceinline__ int ta_step_exponent(float step) {
  return min(max(static_cast<int>((__float_as_uint(step) >> 23) & 255) - 127, TA_STEP_LOW), TA_STEP_HIGH);
}
__device__ __forceinline__ float ta_step_log2(float step) {
  return fminf(fmaxf(__log2f(step), static_cast<float>(TA_STEP_LOW)), static_cast<float>(TA_STEP_HIGH));
}

__device__ __forceinline__ float ta_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D[16x8] += A[16x16] B[16x8], fp32 accumulation (warp-wide)
template <bool BF>
__device__ __forceinline__ void ta_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ta_ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ta_ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t ta_lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ta_lds4f(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ta_lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// 16 bytes (or, with `have` false, 16 zero bytes) into shared memory
__device__ __forceinline__ void ta_copy16(uint32_t dst, const void* src, bool have) {
  const int n = have ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void ta_copy4(uint32_t dst, const void* src, bool have) {
  const int n = have ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void ta_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ta_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t ta_pack(float a, float b, bool bf) {
  if (bf) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four stored 8-bit values as two f16 pairs, exactly.
template <int FMT>
__device__ __forceinline__ void ta_widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == TA_FP8) {
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // byte + 128 becomes the low bits of 1024 + byte + 128; subtract 1152
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __float2half2_rn(1152.0f);
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off), hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  }
}

// Factor of a partial result with reference `ref` and sum `sum` against reference `top`.
// One that saw no key counts nothing; one whose scores were all NaN (its reference never
// moved, its sum is NaN) and one with an infinite score stay in, and give NaN.
__device__ __forceinline__ float ta_share(float ref, float sum, float top) {
  if (ref == -INFINITY) return sum == 0.0f ? 0.0f : 1.0f;
  return ta_exp2(ref - top);
}

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
// (A call has fewer than 2^31 tiles.)
struct TaShare {
  int b, base, u, end;
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
  s.u = static_cast<int>(total * cta / ctas);
  s.end = static_cast<int>(total * (cta + 1) / ctas);
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
    s.base = static_cast<int>(base);
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
  int kvh;                   // the segment's key head
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
    while (s.u >= s.base + tiles * per_seq) {  // (ends: u < end <= all tiles)
      s.base += tiles * per_seq;
      ++s.b;
      load(p, unit);
    }
    const int at = s.u - s.base;
    o.b = s.b;
    o.seg = at / tiles;
    o.t0 = at - o.seg * tiles;
    o.kvh = o.seg / p.row_tiles;
    o.tiles = tiles;
    o.n = min(tiles - o.t0, s.end - s.u);
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

// Asynchronous copies of this thread so far arrive on `bar` when they have landed.
__device__ __forceinline__ void tc_copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}


// ── up to 16 rows per key head ───────────────────────────────────────────────────
// Decoding: every key is read once for a handful of rows, so HBM bounds it, and what a warp
// does for a block of keys must stay below the block's share of that time.  A persistent
// CTA takes an equal run of units (NW blocks of KB keys, a block a warp); a warp keeps its
// own ring of blocks in flight across the parts of the run.  16-bit rows: 16 keys a block,
// cp.async into a swizzled layout for ldmatrix.  8-bit rows: 32 keys a block, one bulk copy
// for each run of a page (a warp's block in one piece, unswizzled: reading it meets a bank
// two to four times, which costs less than permuting copies, about a hundred instructions
// a block), widened to f16 in registers.  mma.sync m16n8k16 with the queries as the 16 rows.
template <int FMT, int D, bool FEW>
struct TaLayout {
  static constexpr bool QUANT = FMT >= TA_INT8;
  static constexpr int ES = QUANT ? 1 : 2;
  static constexpr int KB = QUANT ? 32 : 16;            // keys per block
  static constexpr int CPR = D * ES / 16;               // 16-byte chunks per row
  static constexpr int TILE = KB * D * ES;              // K (or V) bytes per block
  static constexpr int STAGE = 2 * TILE + (QUANT ? KB * 8 : 0);  // 8 bits: (key step, value step) a key
  static constexpr int NW = QUANT && FEW ? 12 : 8;      // warps per CTA
  static constexpr int UNIT = NW * KB;
  static constexpr int ST = D == 128 ? (NW == 12 ? 2 : 3) : 4;  // ring depth
  static constexpr int RING = NW * ST * STAGE;
  static constexpr int MERGE = NW * 4 * (D * 4 + 8);    // four rows of every warp's result at a time
  static constexpr int SMEM = RING + MERGE;
  static_assert(SMEM + 2048 <= 227 * 1024, "shared memory");
};

// Byte offset of 16-byte chunk c of row r of a 16-bit block: eight rows at one chunk lie in
// eight different bank groups.
template <int D>
__device__ __forceinline__ uint32_t ta_chunk(int r, int c) {
  return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

// FEW: at most eight rows, so the fragments' rows 8-15 are empty and their softmax is left out.
template <int FMT, int D, bool FEW>
__global__ void __launch_bounds__(TaLayout<FMT, D, FEW>::NW * 32, 1) tree_attention_kernel(const TaParams p, uint64_t budget) {
  using L = TaLayout<FMT, D, FEW>;
  constexpr bool QUANT = L::QUANT, BF = FMT == TA_BF16;
  constexpr int KB = L::KB, NT = KB / 8, DT = D / 8, KS = D / 16, H = FEW ? 1 : 2, NW = L::NW;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[QUANT ? NW * L::ST : 1];
  __shared__ TaShare s_share;
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rows = p.tokens * p.group;  // row r: token r / group, head r % group
  const int per_seq = p.cache.kv_heads;
  if (threadIdx.x == 0) s_abort = 0;
  if constexpr (QUANT) {
    if (lane < L::ST) mbar_init(smem_u32(&bars[warp * L::ST + lane]), 33);
    fence_mbar_init();
  }
  if (warp == 0) {
    const TaShare s = ta_share_of(p, per_seq, L::UNIT, blockIdx.x, gridDim.x);
    if (lane == 0) s_share = s;
  }
  __syncthreads();
  TaWalk walk;
  walk.begin(p, s_share, L::UNIT);

  // ── blocks in flight ─────────────────────────────────────────────────────────
  const uint32_t ring = smem_u32(smem) + warp * (L::ST * L::STAGE);
  const uint32_t bar = smem_u32(&bars[QUANT ? warp * L::ST : 0]);
  const uint8_t* kbase = static_cast<const uint8_t*>(p.cache.k);
  const uint8_t* vbase = static_cast<const uint8_t*>(p.cache.v);
  TaWalk in_walk = walk;
  TaPart in_part;
  in_part.n = 0;
  int in_unit = 0, in_stage = 0;
  auto fetch = [&]() {
    bool live = true;
    if (in_unit >= in_part.n) {
      in_unit = 0;
      live = in_walk.next(p, per_seq, L::UNIT, in_part);
      if (!live) in_part.n = 0;
    }
    if (live) {
      const int k0 = (in_part.t0 + in_unit) * L::UNIT + warp * KB, hi = in_part.ctx + in_part.drafts;
      const uint32_t dst = ring + in_stage * L::STAGE;
      // lane r < KB finds row k0 + r
      int row = -1, at = 0;
      const int key = k0 + lane;
      if (lane < KB && key < hi) {
        const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.cache.page_size;
        const int id = p.page_table[static_cast<int64_t>(in_part.b) * p.width + pg];
        at = key - pg * p.cache.page_size;
        if (id >= 0 && id < p.cache.num_pages)
          row = (id * p.cache.kv_heads + in_part.kvh) * p.cache.page_size + at;
        else
          index_error();
      }
      if constexpr (!QUANT) {
        constexpr int N = KB * L::CPR / 32;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = lane + 32 * i, r = c / L::CPR, col = c % L::CPR;
          const int rr = __shfl_sync(0xffffffffu, row, r);
          const int64_t off = rr < 0 ? 0 : static_cast<int64_t>(rr) * (D * 2) + col * 16;
          ta_copy16(dst + ta_chunk<D>(r, col), kbase + off, rr >= 0);
          ta_copy16(dst + L::TILE + ta_chunk<D>(r, col), vbase + off, rr >= 0);
        }
      } else {
        const uint32_t full = bar + 8 * in_stage;
        const int len = row >= 0 && (lane == 0 || at == 0) ? min(min(p.cache.page_size - at, KB - lane), hi - key) * D : 0;
        const uint32_t bytes = __reduce_add_sync(0xffffffffu, len);
        if (lane == 0) mbar_arrive_expect_tx(full, 2 * bytes);
        __syncwarp();
        if (len) {
          bulk_load_g2s(dst + lane * D, kbase + static_cast<int64_t>(row) * D, len, full);
          bulk_load_g2s(dst + L::TILE + lane * D, vbase + static_cast<int64_t>(row) * D, len, full);
        }
        ta_copy4(dst + 2 * L::TILE + lane * 8, p.cache.k_scale + max(row, 0), row >= 0);
        ta_copy4(dst + 2 * L::TILE + lane * 8 + 4, p.cache.v_scale + max(row, 0), row >= 0);
        tc_copies_arrive(full);
      }
      ++in_unit;
    }
    if constexpr (!QUANT) ta_commit();
    in_stage = in_stage + 1 == L::ST ? 0 : in_stage + 1;
    return live;
  };
  int issued = 0;  // blocks whose copies were started
#pragma unroll 1
  for (int n = 0; n < L::ST - 1; ++n) issued += fetch();

  float* merge = reinterpret_cast<float*>(smem + L::RING);  // [NW][4][D], then references and sums
  float2* merge_ml = reinterpret_cast<float2*>(merge + NW * 4 * D);
  TaPart part;
  int stage = 0, used = 0;
  uint32_t phase = 0;
  bool ok = true;
  while (walk.next(p, per_seq, L::UNIT, part)) {
    const int b = part.b, kvh = part.kvh, ctx = part.ctx, hi = part.ctx + part.drafts;
    // ── query fragments: rows g and g + 8 ────────────────────────────────────────
    uint32_t qf[KS][4];
    float row_scale[2];
    int token[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = half * 8 + g;
      const int i = r / p.group;
      const bool valid = r < rows && i < part.drafts && half < H;
      token[half] = valid ? i : -1;
      row_scale[half] = p.scale_log2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks][half] = qf[ks][2 + half] = 0;
      if (half >= H) continue;
      const int64_t off = b * p.q_sb + static_cast<int64_t>(valid ? i : 0) * p.q_st +
                          static_cast<int64_t>(kvh * p.group + (valid ? r % p.group : 0)) * p.q_sh;
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + off;
      // 16-bit keys: a step's elements 16 ks + 2 t, + 1, + 8, + 9.  8-bit keys: four
      // neighbours of the 16-byte chunk that the thread reads of a key.
      uint2 raw[KS];
      const bool wide = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && ((p.q_sb | p.q_st | p.q_sh) & 3) == 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        raw[ks] = make_uint2(0, 0);
        if (!valid) continue;
        const int d = QUANT ? 16 * (t + 4 * (ks / 4)) + 4 * (ks % 4) : 16 * ks + 2 * t;
        constexpr int STEP = QUANT ? 2 : 8;
        if (wide) {
          if (QUANT) raw[ks] = *reinterpret_cast<const uint2*>(src + d);
          else raw[ks] = make_uint2(*reinterpret_cast<const uint32_t*>(src + d), *reinterpret_cast<const uint32_t*>(src + d + STEP));
        } else {
          raw[ks].x = src[d] | (static_cast<uint32_t>(src[d + 1]) << 16);
          raw[ks].y = src[d + STEP] | (static_cast<uint32_t>(src[d + STEP + 1]) << 16);
        }
      }
      if constexpr (!QUANT) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qf[ks][half] = raw[ks].x;
          qf[ks][2 + half] = raw[ks].y;
        }
      } else {
        // into f16's range by a power of two
        auto f32 = [&](uint32_t h) {
          return p.dtype == OJX_BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
        };
        float amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          amax = fmaxf(fmaxf(amax, fmaxf(fabsf(f32(raw[ks].x & 0xffffu)), fabsf(f32(raw[ks].x >> 16)))),
                       fmaxf(fabsf(f32(raw[ks].y & 0xffffu)), fabsf(f32(raw[ks].y >> 16))));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        float up = 1.0f;
        if (amax > 0.0f && amax < INFINITY) {
          const int ex = min(max(ilogbf(amax), -100), 100);
          up = exp2f(static_cast<float>(8 - ex));  // exact; |x| * up < 512
          row_scale[half] *= exp2f(static_cast<float>(ex - 8));
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qf[ks][half] = ta_pack(f32(raw[ks].x & 0xffffu) * up, f32(raw[ks].x >> 16) * up, false);
          qf[ks][2 + half] = ta_pack(f32(raw[ks].y & 0xffffu) * up, f32(raw[ks].y >> 16) * up, false);
        }
      }
    }

    float o[DT][4];
    float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

    for (int n = 0; n < part.n; ++n) {
      if constexpr (QUANT) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar + 8 * stage, phase, budget, &s_abort));
      } else {
        ta_wait<L::ST - 2>();
      }
      __syncwarp();
      if (ok) issued += fetch();
      const uint32_t sk = ring + stage * L::STAGE, sv = sk + L::TILE;
      if (ok) {  // (after a wait that ran out: stays at the first block not known to have landed)
        ++used;
        if (++stage == L::ST) stage = 0, phase ^= 1;
      }
      const int k0 = (part.t0 + n) * L::UNIT + warp * KB;
      if (k0 >= hi || !ok) continue;  // uniform
      const bool all = k0 + KB <= ctx;  // no drafts and no end inside this block

      // scores
      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
      if constexpr (!QUANT) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t kb[4];
          const int r = (lane & 7) + ((lane >> 4) << 3);
          ta_ldsm4(sk + ta_chunk<D>(r, 2 * ks + ((lane >> 3) & 1)), kb);
          ta_mma<BF>(s[0], qf[ks], kb[0], kb[1]);
          ta_mma<BF>(s[1], qf[ks], kb[2], kb[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const uint4 w = ta_lds128(sk + (8 * j + g) * D + (t + 4 * i) * 16);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t b0, b1;
              ta_widen4<FMT>(ww[c], b0, b1);
              ta_mma<false>(s[j], qf[4 * i + c], b0, b1);
            }
          }
      }

      // this thread's two keys of each tile: their steps (8 bits)
      float ks2[NT][2], vs2[NT][2], lv[NT][2];
      float above = 0.0f;
      bool narrow = true;
      if constexpr (QUANT) {
        // value steps of one block that lie close together: the largest stands for all
        const float own = k0 + lane < hi ? ld_shared_f32(sk + 2 * L::TILE + lane * 8 + 4) : 0.0f;
        const int e = ta_step_exponent(own);
        const int big = __reduce_max_sync(0xffffffffu, own > 0.0f ? e : -1000);
        const int small = __reduce_min_sync(0xffffffffu, own > 0.0f ? e : 1000);
        narrow = big - small <= TA_NEAR;
        above = static_cast<float>(big > -1000 ? big + 1 : TA_STEP_LOW);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float4 st = ta_lds4f(sk + 2 * L::TILE + (8 * j + 2 * t) * 8);
          ks2[j][0] = st.x, vs2[j][0] = st.y, ks2[j][1] = st.z, vs2[j][1] = st.w;
#pragma unroll
          for (int c = 0; c < 2; ++c) lv[j][c] = narrow ? above : ta_step_log2(vs2[j][c]);
        }
      }

      // bit 2 j + e: the keys that this thread's rows see
      uint32_t seen[2] = {token[0] < 0 ? 0u : 0xffffffffu, token[1] < 0 ? 0u : 0xffffffffu};
      if (!all) {
#pragma unroll
        for (int half = 0; half < H; ++half) {
          const uint32_t bits = ta_visible(p, b, token[half], k0, ctx, hi);
          seen[half] = 0;
#pragma unroll
          for (int j = 0; j < NT; ++j) seen[half] |= ((bits >> (8 * j + 2 * t)) & 3u) << (2 * j);
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2 * H; ++e) {
          const int half = e >> 1;
          s[j][e] *= QUANT ? row_scale[half] * ks2[j][e & 1] : row_scale[half];
          if ((seen[half] >> (2 * j + (e & 1))) & 1) top[half] = fmaxf(top[half], QUANT ? s[j][e] + lv[j][e & 1] : s[j][e]);
        }
      float use[2] = {0.0f, 0.0f};
#pragma unroll
      for (int half = 0; half < H; ++half) {
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
        if (!BF) top[half] -= TA_BIAS;
        // the reference moves only when a weight would pass 2^15 (bf16: 2^8), so o is seldom rescaled
        const bool raise = top[half] > ref[half] + 8.0f;
        const float next = raise ? top[half] : ref[half];
        use[half] = next == -INFINITY ? 0.0f : next;
        if (__any_sync(0xffffffffu, raise)) {
          const float alpha = raise ? ta_exp2(ref[half] - use[half]) : 1.0f;
          sum[half] *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            o[d][2 * half] *= alpha;
            o[d][2 * half + 1] *= alpha;
          }
        }
        ref[half] = next;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          if (half >= H) {
            s[j][e] = 0.0f;
            continue;
          }
          const float w = ta_exp2(s[j][e] - use[half]);
          const bool v = (seen[half] >> (2 * j + (e & 1))) & 1;
          sum[half] += v ? w : 0.0f;
          s[j][e] = v ? (QUANT ? w * vs2[j][e & 1] : w) : 0.0f;
        }

      // o += weights * values, 16 keys at a time
      bool odd_v = false;
#pragma unroll
      for (int kk = 0; kk < KB / 16; ++kk) {
        uint32_t pa[4], pl[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float* c = &s[2 * kk + (q >> 1)][2 * (q & 1)];
          pa[q] = ta_pack(c[0], c[1], BF);
          if constexpr (BF) {  // the weight's next eight bits: bf16 alone would double the output's rounding
            const __nv_bfloat162 hi2 = *reinterpret_cast<const __nv_bfloat162*>(&pa[q]);
            pl[q] = ta_pack(c[0] - __low2float(hi2), c[1] - __high2float(hi2), true);
          }
        }
#pragma unroll
        for (int dd = 0; dd < (QUANT ? D / 32 : D / 16); ++dd) {
          constexpr int TN = QUANT ? 4 : 2;  // output tiles fed by one read
          uint32_t vb[TN][2];
          if constexpr (!QUANT) {
            uint32_t x[4];
            const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
            ta_ldsm4_t(sv + ta_chunk<D>(r, 2 * dd + (lane >> 4)), x);
            vb[0][0] = x[0], vb[0][1] = x[1], vb[1][0] = x[2], vb[1][1] = x[3];
          } else {
            // tile c of this read holds columns 32 dd + 4 g + c, so one word serves four tiles
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int r = 16 * kk + 2 * t + (q & 1) + 8 * (q >> 1);
              w[q] = ta_lds32(sv + r * D + 32 * dd + 4 * g);
              if (!all && k0 + r >= hi) w[q] = 0;  // past the end the ring holds an older block
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint32_t u = __byte_perm(w[2 * q], w[2 * q + 1], 0x5140);  // columns 0, 1 of both rows
              const uint32_t v = __byte_perm(w[2 * q], w[2 * q + 1], 0x7362);  // columns 2, 3
              ta_widen4<FMT>(u, vb[0][q], vb[1][q]);
              ta_widen4<FMT>(v, vb[2][q], vb[3][q]);
            }
          }
          if (FMT != TA_INT8 && !all) {
            // a hidden key's NaN or infinity must not reach a row through 0 * value: take it
            // out here, and give it to the rows that do see it below
            constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int c = 0; c < TN; ++c)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                if ((vb[c][q] & EXP) == EXP) vb[c][q] &= 0xffff0000u, odd_v = true;
                if (((vb[c][q] >> 16) & EXP) == EXP) vb[c][q] &= 0x0000ffffu, odd_v = true;
              }
          }
#pragma unroll
          for (int c = 0; c < TN; ++c) {
            ta_mma<BF>(o[TN * dd + c], pa, vb[c][0], vb[c][1]);
            if constexpr (BF) ta_mma<BF>(o[TN * dd + c], pl, vb[c][0], vb[c][1]);
          }
        }
      }
      if (FMT != TA_INT8 && __any_sync(0xffffffffu, odd_v)) {
        for (int r = 0; r < KB; ++r) {
          if (k0 + r >= hi) break;
#pragma unroll
          for (int half = 0; half < H; ++half) {
            if (!(ta_visible(p, b, token[half], k0 + r, ctx, hi) & 1)) continue;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                // column of o[dt][2 half + e] (see the value reads above)
                const int col = QUANT ? 32 * (dt / 4) + 4 * (2 * t + e) + dt % 4 : 8 * dt + 2 * t + e;
                const uint32_t a = QUANT ? sv + r * D + col : sv + ta_chunk<D>(r, col / 8) + (col % 8) * 2;
                const uint32_t word = ta_lds32(a & ~3u) >> (8 * (a & 3));
                float v;
                if constexpr (QUANT) {
                  uint32_t h, unused;
                  ta_widen4<FMT>(word & 0xffu, h, unused);
                  v = __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
                } else if constexpr (BF) {
                  v = __uint_as_float(word << 16);
                } else {
                  v = __half2float(__ushort_as_half(static_cast<unsigned short>(word & 0xffffu)));
                }
                if (!(fabsf(v) < INFINITY)) o[dt][2 * half + e] += v;
              }
          }
        }
      }
      __syncwarp();
    }

    // ── join the warps, four rows at a time ────────────────────────────────────────
#pragma unroll
    for (int half = 0; half < H; ++half) {
      sum[half] += __shfl_xor_sync(0xffffffffu, sum[half], 1);
      sum[half] += __shfl_xor_sync(0xffffffffu, sum[half], 2);
    }
    const bool whole = part.n == part.tiles;
#pragma unroll
    for (int c = 0; c < 2 * H; ++c) {  // rows 4 c .. 4 c + 3
      if (4 * c >= rows) break;        // uniform
      constexpr int R = 4;
      if ((g >> 2) == (c & 1)) {
        const int half = c >> 1;
        if (t == 0) merge_ml[warp * R + (g & 3)] = make_float2(ref[half], sum[half]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = QUANT ? 32 * (dt / 4) + 4 * (2 * t + e) + dt % 4 : 8 * dt + 2 * t + e;
            merge[(warp * R + (g & 3)) * D + col] = o[dt][2 * half + e];
          }
      }
      __syncthreads();
      for (int x = threadIdx.x; x < R * D; x += NW * 32) {
        const int r = x / D, d = x % D, gr = 4 * c + r;
        if (gr >= rows) break;
        float2 ml[NW];
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          ml[w] = merge_ml[w * R + r];
          top = fmaxf(top, ml[w].x);
        }
        float acc = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float f = ta_share(ml[w].x, ml[w].y, top);
          if (f != 0.0f) {
            acc += f * merge[(w * R + r) * D + d];
            l += f * ml[w].y;
          }
        }
        if (whole) {
          const int64_t at = ((static_cast<int64_t>(b) * p.tokens + gr / p.group) * p.q_heads + kvh * p.group + gr % p.group) * D + d;
          store_as(p.out, at, p.dtype, l == 0.0f ? 0.0f : acc / l);
        } else {
          const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (part.first ? 0 : 1)) * 16 + gr;
          p.part_o[slot * D + d] = acc;
          if (d == 0) p.part_ml[slot] = make_float2(top, l);
        }
      }
      __syncthreads();
    }
  }
  grid_dep_launch_dependents();  // the join kernel may start; it waits for this grid's end
  if constexpr (QUANT) {
    // (after a wait that ran out: let the copies in flight land before the CTA may exit)
    for (; used < issued; ++used) {
      mbar_wait_drain(bar + 8 * stage, phase, budget);
      if (++stage == L::ST) stage = 0, phase ^= 1;
    }
  } else {
    ta_wait<0>();
  }
}

// Joins the parts of segments that more than one CTA took, and writes the zeros of
// sequences without keys.  One warp per row; the parts' factors sit in the lanes, so the
// loads of a pass over 32 parts do not wait for one another.  It starts while the attention
// kernel ends (batch of 64: 191 -> 183 us a call) and takes about 5 us, most of it latency.
template <int D>
__global__ void __launch_bounds__(128) tree_attention_parts_kernel(const TaParams p, int tile_rows, int unit, int ctas) {
  constexpr int E = D / 32;  // values a lane
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
  grid_dep_wait();  // the parts are written (all above reads the call's inputs only)
  const int64_t at = ((static_cast<int64_t>(b) * p.tokens + r / p.group) * p.q_heads + kvh * p.group + r % p.group) * D;
  if (tiles == 0) {
    for (int i = 0; i < E; ++i) store_as(p.out, at + lane * E + i, p.dtype, 0.0f);
    return;
  }
  // CTA c's first tile, total * c / ctas, with one long division for all; and the CTA that has tile u.
  const long long all = total * per_seq, each = all / ctas;
  const int rest = static_cast<int>(all - each * ctas);
  auto first_of = [&](int c) { return each * c + rest * c / ctas; };
  auto owner = [&](long long u) {
    int c = min(static_cast<int>(static_cast<float>(u) * (static_cast<float>(ctas) / static_cast<float>(all))), ctas - 1);
    while (first_of(c) > u) --c;
    while (c + 1 < ctas && first_of(c + 1) <= u) ++c;
    return c;
  };
  const long long u0 = before * per_seq + (kvh * p.row_tiles + r / tile_rows) * tiles;
  const int c0 = owner(u0), c1 = owner(u0 + tiles - 1);
  if (c0 == c1) return;  // written by its CTA
  const bool first0 = first_of(c0) == u0;
  auto slot_of = [&](int c) {
    return (static_cast<int64_t>(c) * 2 + (c > c0 || first0 ? 0 : 1)) * tile_rows + r % tile_rows;
  };
  float ref = -INFINITY, acc[E], l = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.0f;
  for (int c = c0; c <= c1; c += 32) {
    const int mine = c + lane;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (mine <= c1 && first_of(mine) < first_of(mine + 1)) ml = p.part_ml[slot_of(mine)];  // (or no tiles)
    float top = fmaxf(ref, ml.x);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float keep = ta_share(ref, l, top), f = ta_share(ml.x, ml.y, top);
    float part = f != 0.0f ? f * ml.y : 0.0f;
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    l = (keep != 0.0f ? l * keep : 0.0f) + part;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = keep != 0.0f ? acc[i] * keep : 0.0f;
    ref = top;
    const int n = min(32, c1 - c + 1);
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float g = __shfl_sync(0xffffffffu, f, k);
      float o[E];
      if constexpr (E == 4) {
        *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(p.part_o + slot_of(c + k) * D + lane * E);
      } else {
        *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(p.part_o + slot_of(c + k) * D + lane * E);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] += g != 0.0f ? g * o[i] : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) store_as(p.out, at + lane * E + i, p.dtype, l == 0.0f ? 0.0f : acc[i] / l);
}

}  // namespace ojx
