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
// For the values the step joins the weight: sum_j (p_j step_vj) v8_j.  The weights of a row
// are kept below one by measuring them against the largest s_j + log2(step_vj) instead of
// the largest s_j, so they use f16's range whatever the steps are.  A bf16 query row is
// brought into f16's range by a power of two, which the score's factor takes back.
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
  int row_tiles, splits;
  int page_shift;  // log2 of the page size, or -1
  int box_rows;    // rows of a TMA box (16-bit caches on tcgen05), 0: no TMA
  float* part_o;   // [segment][split][rows][D], unnormalised
  float2* part_ml;  // [segment][split][rows]: reference, sum
};

constexpr int TA_F16 = 0, TA_BF16 = 1, TA_INT8 = 2, TA_FP8 = 3;

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

template <int FMT, int D, int MT>
struct TaLayout {
  static constexpr bool QUANT = FMT >= TA_INT8;
  static constexpr int ES = QUANT ? 1 : 2;
  static constexpr int KB = QUANT ? 32 : 16;            // keys per warp step
  static constexpr int CPR = D * ES / 16;               // 16-byte chunks per row
  static constexpr int TILE = KB * D * ES;              // K (or V) bytes per step
  static constexpr int STAGE = 2 * TILE + (QUANT ? 2 * KB * 4 : 0);
  static constexpr int NW = 8;                          // warps per block
  static constexpr int ST = D == 128 ? 3 : 4;           // ring depth
  static constexpr int ROWS = 16 * MT;
  static constexpr int RING = NW * ST * STAGE;
  static constexpr int MERGE = NW * ROWS * (D * 4 + 8);  // the warps' partial results, after the loop
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Shared-memory byte offset of 16-byte chunk c of row r: the swizzles keep the fragment
// reads below free of bank conflicts (16-bit rows: eight rows at one chunk; 8-bit keys:
// two rows x four chunks; 8-bit values: rows 2t, t < 4, at one 32-byte granule).
template <int FMT, int D, bool IS_V>
__device__ __forceinline__ uint32_t ta_chunk(int r, int c) {
  if constexpr (FMT < TA_INT8) return r * (D * 2) + ((c ^ (r & 7)) << 4);
  if constexpr (!IS_V) return D == 128 ? r * 128 + ((c ^ ((r & 1) << 2)) << 4) : r * 64 + (c << 4);
  if constexpr (D == 128) return r * 128 + ((c ^ (((r >> 1) & 3) << 1)) << 4);
  const int line = r >> 1, in = ((r & 1) << 2) | c;  // two 64-byte rows per line
  return line * 128 + ((in ^ ((line & 3) << 1)) << 4);
}

template <int FMT, int D, int MT>
__global__ void __launch_bounds__(TaLayout<FMT, D, MT>::NW * 32, 1) tree_attention_kernel(const TaParams p) {
  using L = TaLayout<FMT, D, MT>;
  constexpr bool QUANT = L::QUANT, BF = FMT == TA_BF16;
  constexpr int KB = L::KB, NT = KB / 8, DT = D / 8, KS = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;

  int seg = blockIdx.x / p.splits;
  const int split = blockIdx.x % p.splits;
  const int rt = seg % p.row_tiles;
  const int kvh = (seg / p.row_tiles) % p.cache.kv_heads;
  const int b = seg / (p.row_tiles * p.cache.kv_heads);
  const int rows = p.tokens * p.group;  // row r: token r / group, head r % group

  int ctx = max(p.contexts[b], 0);
  int drafts = p.drafts ? min(max(p.drafts[b], 0), p.tokens) : p.tokens;
  const int64_t room = static_cast<int64_t>(p.width) * p.cache.page_size;
  if (static_cast<int64_t>(ctx) + drafts > room) {  // more keys than the page table holds
    if (threadIdx.x == 0) index_error();
    ctx = static_cast<int>(min(static_cast<int64_t>(ctx), room));
    drafts = static_cast<int>(min(static_cast<int64_t>(drafts), room - ctx));
  }
  const int keys = ctx + drafts;
  constexpr int STEP = L::NW * KB;
  const int per = ((keys + p.splits - 1) / p.splits + STEP - 1) / STEP * STEP;
  const int lo = min(keys, split * per), hi = min(keys, lo + per);

  // ── query fragments: rows g and g + 8 of each 16-row tile ────────────────────
  uint32_t qf[MT][KS][4];
  float row_scale[MT][2];
  int token[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = rt * L::ROWS + m * 16 + half * 8 + g;
      const int i = r / p.group;
      const bool valid = r < rows && i < drafts;
      token[m][half] = valid ? i : -1;
      const int64_t off = b * p.q_sb + static_cast<int64_t>(valid ? i : 0) * p.q_st +
                          static_cast<int64_t>(kvh * p.group + (valid ? r % p.group : 0)) * p.q_sh;
      float x[KS * 4];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // 16-bit keys: the fragment's own order; 8-bit keys: a thread's four elements of a
          // step are four neighbours of the 16-byte chunk it reads
          const int d = QUANT ? 16 * (t + 4 * (ks / 4)) + 4 * (ks % 4) + e : 16 * ks + 2 * t + (e & 1) + 8 * (e >> 1);
          const float v = !valid ? 0.0f
                          : p.dtype == OJX_BF16
                              ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[off + d])
                              : __half2float(static_cast<const __half*>(p.q)[off + d]);
          x[ks * 4 + e] = v;
        }
      float back = 1.0f;
      if (QUANT) {
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < KS * 4; ++e) amax = fmaxf(amax, fabsf(x[e]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        if (amax > 0.0f && amax < INFINITY) {
          const int ex = min(max(ilogbf(amax), -100), 100);
          const float up = exp2f(static_cast<float>(8 - ex));  // exact; |x| * up < 512
          back = exp2f(static_cast<float>(ex - 8));
#pragma unroll
          for (int e = 0; e < KS * 4; ++e) x[e] *= up;
        }
      }
      row_scale[m][half] = p.scale_log2 * back;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[m][ks][half] = ta_pack(x[ks * 4], x[ks * 4 + 1], BF);
        qf[m][ks][2 + half] = ta_pack(x[ks * 4 + 2], x[ks * 4 + 3], BF);
      }
    }

  float o[MT][DT][4];
  float ref[MT][2], sum[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][n][e] = 0.0f;
    ref[m][0] = ref[m][1] = -INFINITY;
    sum[m][0] = sum[m][1] = 0.0f;
  }

  // ── key blocks of this warp: lo + (n * NW + warp) * KB ─────────────────────────
  const uint32_t ring = smem_u32(smem) + warp * (L::ST * L::STAGE);
  const int32_t* table = p.page_table + static_cast<int64_t>(b) * p.width;
  const int first = lo + warp * KB;
  const int blocks = first < hi ? (hi - first + STEP - 1) / STEP : 0;
  const uint8_t* kbase = static_cast<const uint8_t*>(p.cache.k);
  const uint8_t* vbase = static_cast<const uint8_t*>(p.cache.v);
  auto fetch = [&](int n) {
    if (n < blocks) {
      const int k0 = first + n * STEP;
      const uint32_t dst = ring + (n % L::ST) * L::STAGE;
      // lane r < KB finds row k0 + r once; the copies get it by shuffle
      long long row = -1;
      const int key = k0 + lane;
      if (lane < KB && key < hi) {
        const int pg = key / p.cache.page_size;
        const int id = table[pg];
        if (id >= 0 && id < p.cache.num_pages)
          row = (static_cast<long long>(id) * p.cache.kv_heads + kvh) * p.cache.page_size + (key - pg * p.cache.page_size);
        else
          index_error();
      }
      constexpr int N = KB * L::CPR / 32;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = lane + 32 * i, r = c / L::CPR, col = c % L::CPR;
        const long long rr = __shfl_sync(0xffffffffu, row, r);
        const int64_t off = rr < 0 ? 0 : rr * (D * L::ES) + col * 16;
        ta_copy16(dst + ta_chunk<FMT, D, false>(r, col), kbase + off, rr >= 0);
        ta_copy16(dst + L::TILE + ta_chunk<FMT, D, true>(r, col), vbase + off, rr >= 0);
      }
      if constexpr (QUANT) {
        ta_copy4(dst + 2 * L::TILE + lane * 4, p.cache.k_scale + (row < 0 ? 0 : row), row >= 0);
        ta_copy4(dst + 2 * L::TILE + KB * 4 + lane * 4, p.cache.v_scale + (row < 0 ? 0 : row), row >= 0);
      }
    }
    ta_commit();
  };
#pragma unroll
  for (int n = 0; n < L::ST - 1; ++n) fetch(n);

  for (int n = 0; n < blocks; ++n) {
    ta_wait<L::ST - 2>();
    __syncwarp();
    fetch(n + L::ST - 1);
    const uint32_t sk = ring + (n % L::ST) * L::STAGE, sv = sk + L::TILE;
    const int k0 = first + n * STEP;

    // scores
    float s[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][j][e] = 0.0f;
    if constexpr (!QUANT) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kb[4];
        const int r = (lane & 7) + ((lane >> 4) << 3);
        ta_ldsm4(sk + ta_chunk<FMT, D, false>(r, 2 * ks + ((lane >> 3) & 1)), kb);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          ta_mma<BF>(s[m][0], qf[m][ks], kb[0], kb[1]);
          ta_mma<BF>(s[m][1], qf[m][ks], kb[2], kb[3]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint4 w = ta_lds128(sk + ta_chunk<FMT, D, false>(8 * j + g, t + 4 * i));
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t b0, b1;
            ta_widen4<FMT>(ww[c], b0, b1);
#pragma unroll
            for (int m = 0; m < MT; ++m) ta_mma<false>(s[m][j], qf[m][4 * i + c], b0, b1);
          }
        }
    }

    // a key's step and reference offset, for this thread's two columns of each tile
    float ks2[NT][2], vs2[NT][2], lv[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ks2[j][e] = vs2[j][e] = 1.0f;
        lv[j][e] = 0.0f;
        if constexpr (QUANT) {
          const uint32_t a = sk + 2 * L::TILE + (8 * j + 2 * t + e) * 4;
          ks2[j][e] = ld_shared_f32(a);
          vs2[j][e] = ld_shared_f32(a + KB * 4);
          // clamped, so that p = w / step stays far inside fp32's range
          lv[j][e] = fminf(fmaxf(__log2f(vs2[j][e]), -60.0f), 60.0f);
        }
      }

    const bool all = k0 + KB <= ctx;  // no drafts and no end inside this block
    bool odd_v = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      // bit 2 j + e: this thread's columns
      uint32_t seen[2] = {token[m][0] < 0 ? 0u : 0xffffffffu, token[m][1] < 0 ? 0u : 0xffffffffu};
      if (!all) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t bits = 0;
          const int i = token[m][half];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = k0 + 8 * j + 2 * t + e, d = key - ctx;
              bool v = i >= 0 && key < hi;
              if (v && d >= 0)
                v = p.mask ? (p.mask[b * p.mask_sb + static_cast<int64_t>(i) * p.words + (d >> 6)] >> (d & 63)) & 1
                           : d <= i;
              bits |= static_cast<uint32_t>(v) << (2 * j + e);
            }
          seen[half] = bits;
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          s[m][j][e] *= QUANT ? row_scale[m][half] * ks2[j][e & 1] : row_scale[m][half];
          if ((seen[half] >> (2 * j + (e & 1))) & 1) top[half] = fmaxf(top[half], s[m][j][e] + lv[j][e & 1]);
        }
      float use[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
        top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
        // the reference moves only when a weight would pass 2^8, so o is seldom rescaled
        const bool raise = top[half] > ref[m][half] + 8.0f;
        const float next = raise ? top[half] : ref[m][half];
        use[half] = next == -INFINITY ? 0.0f : next;
        if (__any_sync(0xffffffffu, raise)) {
          const float alpha = raise ? ta_exp2(ref[m][half] - use[half]) : 1.0f;
          sum[m][half] *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            o[m][d][2 * half] *= alpha;
            o[m][d][2 * half + 1] *= alpha;
          }
        }
        ref[m][half] = next;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          const float w = ta_exp2(s[m][j][e] - use[half]);
          const bool v = (seen[half] >> (2 * j + (e & 1))) & 1;
          sum[m][half] += v ? w : 0.0f;
          s[m][j][e] = v ? (QUANT ? w * vs2[j][e & 1] : w) : 0.0f;
        }
    }

    // o += weights * values, 16 keys at a time
#pragma unroll
    for (int kk = 0; kk < KB / 16; ++kk) {
      uint32_t pa[MT][4], pl[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float* c = &s[m][2 * kk + (q >> 1)][2 * (q & 1)];
          pa[m][q] = ta_pack(c[0], c[1], BF);
          if constexpr (BF) {  // the weight's next eight bits: bf16 alone would double the output's rounding
            const __nv_bfloat162 hi2 = *reinterpret_cast<const __nv_bfloat162*>(&pa[m][q]);
            pl[m][q] = ta_pack(c[0] - __low2float(hi2), c[1] - __high2float(hi2), true);
          }
        }
#pragma unroll
      for (int dd = 0; dd < (QUANT ? D / 32 : D / 16); ++dd) {
        constexpr int TN = QUANT ? 4 : 2;  // output tiles fed by one read
        uint32_t vb[TN][2];
        if constexpr (!QUANT) {
          uint32_t x[4];
          const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
          ta_ldsm4_t(sv + ta_chunk<FMT, D, true>(r, 2 * dd + (lane >> 4)), x);
          vb[0][0] = x[0], vb[0][1] = x[1], vb[1][0] = x[2], vb[1][1] = x[3];
        } else {
          // tile c of this read holds columns 32 dd + 4 g + c, so one word serves four tiles
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = 16 * kk + 2 * t + (q & 1) + 8 * (q >> 1);
            w[q] = ta_lds32(sv + ta_chunk<FMT, D, true>(r, 2 * dd + (g >> 2)) + (g & 3) * 4);
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
        for (int c = 0; c < TN; ++c)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            ta_mma<BF>(o[m][TN * dd + c], pa[m], vb[c][0], vb[c][1]);
            if constexpr (BF) ta_mma<BF>(o[m][TN * dd + c], pl[m], vb[c][0], vb[c][1]);
          }
      }
    }
    if (FMT != TA_INT8 && __any_sync(0xffffffffu, odd_v)) {
      for (int r = 0; r < KB; ++r) {
        const int key = k0 + r, d = key - ctx;
        if (key >= hi) break;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int i = token[m][half];
            if (i < 0) continue;
            if (d >= 0 && !(p.mask ? (p.mask[b * p.mask_sb + static_cast<int64_t>(i) * p.words + (d >> 6)] >> (d & 63)) & 1
                                   : d <= i))
              continue;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                // column of o[m][dt][2 half + e] (see the value reads above)
                const int col = QUANT ? 32 * (dt / 4) + 4 * (2 * t + e) + dt % 4 : 8 * dt + 2 * t + e;
                const uint32_t a = sv + ta_chunk<FMT, D, true>(r, col * L::ES / 16) + (col * L::ES) % 16;
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
                if (!(fabsf(v) < INFINITY)) o[m][dt][2 * half + e] += v;
              }
          }
      }
    }
    __syncwarp();
  }
  ta_wait<0>();
  __syncthreads();

  // ── join the warps: each writes its sums, reference and o, then all threads add ────
  float* so = reinterpret_cast<float*>(smem);
  float* sref = so + L::NW * L::ROWS * D;
  float* ssum = sref + L::NW * L::ROWS;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float v = sum[m][half];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int r = m * 16 + half * 8 + g;
      if (t == 0) {
        sref[warp * L::ROWS + r] = ref[m][half];
        ssum[warp * L::ROWS + r] = v;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = QUANT ? 32 * (dt / 4) + 4 * (2 * t + e) + dt % 4 : 8 * dt + 2 * t + e;
          so[(warp * L::ROWS + r) * D + col] = o[m][dt][2 * half + e];
        }
    }
  __syncthreads();
  for (int x = threadIdx.x; x < L::ROWS * D; x += blockDim.x) {
    const int r = x / D, d = x % D;
    const int gr = rt * L::ROWS + r;
    if (gr >= rows) break;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < L::NW; ++w) top = fmaxf(top, sref[w * L::ROWS + r]);
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < L::NW; ++w) {
      const float f = ta_share(sref[w * L::ROWS + r], ssum[w * L::ROWS + r], top);
      if (f != 0.0f) {
        acc += f * so[(w * L::ROWS + r) * D + d];
        l += f * ssum[w * L::ROWS + r];
      }
    }
    if (p.splits == 1) {
      const float v = l == 0.0f ? 0.0f : acc / l;
      const int64_t at = ((static_cast<int64_t>(b) * p.tokens + gr / p.group) * p.q_heads + kvh * p.group + gr % p.group) * D + d;
      store_as(p.out, at, p.dtype, v);
    } else {
      const int64_t slot = (static_cast<int64_t>(seg) * p.splits + split) * L::ROWS + r;
      p.part_o[slot * D + d] = acc;
      if (d == 0) p.part_ml[slot] = make_float2(top, l);
    }
  }
}

// Joins the splits of a row: one warp per row.
template <int D>
__global__ void __launch_bounds__(128) tree_attention_join_kernel(const TaParams p, int rows_per_tile) {
  const int lane = threadIdx.x & 31;
  const int rows = p.tokens * p.group;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= static_cast<int64_t>(p.batch) * p.cache.kv_heads * rows) return;
  const int r = static_cast<int>(w % rows);
  const int64_t bh = w / rows;
  const int64_t seg = bh * p.row_tiles + r / rows_per_tile;
  const int64_t slot0 = seg * p.splits * rows_per_tile + r % rows_per_tile;
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, p.part_ml[slot0 + static_cast<int64_t>(s) * rows_per_tile].x);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float acc[D / 32], l = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
  for (int s = 0; s < p.splits; ++s) {
    const int64_t slot = slot0 + static_cast<int64_t>(s) * rows_per_tile;
    const float2 ml = p.part_ml[slot];
    const float f = ta_share(ml.x, ml.y, top);
    if (f != 0.0f) {
      l += f * ml.y;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] += f * p.part_o[slot * D + lane + 32 * i];
    }
  }
  const int b = static_cast<int>(bh / p.cache.kv_heads), kvh = static_cast<int>(bh % p.cache.kv_heads);
  const int64_t at = ((static_cast<int64_t>(b) * p.tokens + r / p.group) * p.q_heads + kvh * p.group + r % p.group) * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_as(p.out, at + lane + 32 * i, p.dtype, l == 0.0f ? 0.0f : acc[i] / l);
}

}  // namespace ojx
