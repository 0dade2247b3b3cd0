// qk_cache.cuh — row kernels of the serving operators: RMS norm of each query and key
// head with the position rotation (forward and gradient), quantisation of key and value
// rows into a paged cache, reading them back, and moving the rows of an accepted path.
//
// A row is one head of one token, D elements.  With c, s the cosine and sine of the
// token's position for pair i, and pairs (a, b) = (i, i + rotary/2) or (2i, 2i + 1):
//   n  = w * x / sqrt(mean(x^2) + eps)
//   y_a = n_a c - n_b s,   y_b = n_a s + n_b c        (elements past rotary: y = n)
// and for dL/dy = g, with h = w * (g turned back by -angle) and r = 1/sqrt(mean(x^2) + eps):
//   dx = r h - x r^3 mean(h x),   dw = sum over rows of (g turned back) * x * r.
// A quantised row keeps step = max|x| * (1/top) in fp32 and round(x / step) in 8 bits
// (top: 127 for int8, 448 for e4m3); a row with a NaN or an infinity reads back as NaN.
//
// Every byte is used once, so these kernels are bound by HBM (a few rows: by latency).
// A lane holds eight elements (where rows are no whole 16-byte vectors: one, several times)
// of both halves of a pair, so the rotation needs no exchange between lanes, and
// 32 / lanes-per-row rows share a warp.
#pragma once
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include "internal.h"
#include "sm100.cuh"

namespace ojx {

// Bit 2 of the device error word: an index given on the device (slot, page, position,
// token, parent) lies outside its range.  The access is skipped.
constexpr unsigned int OJX_DEVERR_INDEX = 4u;

__device__ __forceinline__ void index_error() { atomicOr(&g_dev_error, OJX_DEVERR_INDEX); }

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// One element, and eight (16-byte vectors, p 16-byte aligned), of memory whose type is only
// known at run time (weights).
__device__ __forceinline__ float load_as(const void* p, int64_t at, int dtype) {
  if (dtype == OJX_F32) return static_cast<const float*>(p)[at];
  if (dtype == OJX_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[at]);
  return to_f32(static_cast<const __half*>(p)[at]);
}
template <typename T>
__device__ __forceinline__ void load_eight(const T* p, float (&v)[8]) {
  constexpr int NV = 8 * sizeof(T) / 16;
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
  const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
}
__device__ __forceinline__ void load_eight_as(const void* p, int64_t at, int dtype, float (&v)[8]) {
  if (dtype == OJX_F32) load_eight(static_cast<const float*>(p) + at, v);
  else if (dtype == OJX_BF16) load_eight(static_cast<const __nv_bfloat16*>(p) + at, v);
  else load_eight(static_cast<const __half*>(p) + at, v);
}

__device__ __forceinline__ uint8_t quantise_one(float x, float step, int format) {
  // step 0 (an all-zero row) and a step that is not finite both store zeros; the
  // latter reads back as 0 * step = NaN.
  if (!(step > 0.0f) || step == INFINITY) return 0;
  const float q = x / step;
  if (format == OJX_KV_INT8) {
    const int r = __float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f));
    return static_cast<uint8_t>(static_cast<int8_t>(r));
  }
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ float quantise_step(float amax, int format) {
  return __fmul_rn(amax, format == OJX_KV_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f);
}
__device__ __forceinline__ float dequantise_one(uint8_t b, float step, int format) {
  if (format == OJX_KV_INT8) return static_cast<float>(static_cast<int8_t>(b)) * step;
  const __half_raw h = __nv_cvt_fp8_to_halfraw(b, __NV_E4M3);
  return __half2float(__half(h)) * step;
}
// Larger magnitude, with NaN winning over any number.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct QkParams {
  int64_t tokens;
  int D, rotary, half, npairs, lanes, norm;
  int hq, hk, hv, blocks_per_token, iters;
  int gq, gk, gv;  // row groups (of 32 / lanes heads) of each side
  int dtype_w, pos64, slot64, k_to_cache;
  float eps, inv_dim;
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const void *qw, *kw;
  const float* table;
  int64_t table_rows;
  const void* positions;
  void *q_out, *k_out;
  ojx_kv_cache cache;
  const void* slots;
  // gradient
  const void *gq_data, *gk_data;
  int64_t gq_st, gq_sh, gk_st, gk_sh;
  void *dq, *dk;
  float* partial;  // [blocks][D] sums of dw: q_blocks of the query weight, then the key's
  int q_blocks;
};

// First elements of pair chunk `pi`'s two halves, and whether the pair turns.
template <int CH, bool INTER>
__device__ __forceinline__ bool pair_at(const QkParams& p, int pi, int& a, int& b) {
  if (INTER) {
    a = 2 * pi * CH;
    b = a + CH;
    return a < p.rotary;
  }
  const int turning = p.half / CH;
  if (pi < turning) {
    a = pi * CH;
    b = p.half + a;
    return true;
  }
  a = p.rotary + 2 * (pi - turning) * CH;
  b = a + CH;
  return false;
}

// Cosine and sine of the pair whose first element is `a`.
template <bool INTER>
__device__ __forceinline__ void load_turn(const QkParams& p, int64_t pos, int a, float& cs, float& sn) {
  const float* row = p.table + pos * p.rotary + (INTER ? a / 2 : a);
  cs = row[0];
  sn = row[p.half];
}

// Turn a pair by the angle (sign = 1) or back (sign = -1).
__device__ __forceinline__ void turn_pair(float& xa, float& xb, float cs, float sn, float sign) {
  const float u = xa, v = xb, s = sign * sn;
  xa = u * cs - v * s;
  xb = u * s + v * cs;
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Page row of a slot, or -1 for a slot to skip (negative) or out of range (reported).
__device__ __forceinline__ int64_t slot_row(const ojx_kv_cache& c, int64_t slot, int head) {
  if (slot < 0) return -1;
  const int64_t page = slot / c.page_size;
  if (page >= c.num_pages) {
    index_error();
    return -1;
  }
  return (page * c.kv_heads + head) * c.page_size + slot % c.page_size;
}

__device__ __forceinline__ void store_cached(void* base, int64_t at, int format, float step, float v) {
  if (format == OJX_KV_BF16) static_cast<__nv_bfloat16*>(base)[at] = from_f32<__nv_bfloat16>(v);
  else if (format == OJX_KV_F16) static_cast<__half*>(base)[at] = from_f32<__half>(v);
  else static_cast<uint8_t*>(base)[at] = quantise_one(v, step, format);
}

// Forward rows: query and key heads are normed and rotated (p.norm) and stored densely
// or, keys with k_to_cache and all value heads, into the cache.  A warp takes one token
// and p.iters row groups of it, so the token's cosines are loaded once for its heads.
// For rows that are no whole 16-byte vectors: element loads, whose instructions bound it
// (4096 tokens of 40 heads of 100, bf16: 68 us, 0.97 TB/s).
template <typename T, int NP, bool INTER>
__global__ void __launch_bounds__(256) qk_rows_kernel(const QkParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  const int64_t token = item / p.blocks_per_token;
  if (token >= p.tokens) return;  // whole warp
  const int heads = p.hq + p.hk + p.hv;
  int head = static_cast<int>(item % p.blocks_per_token) * per_warp * p.iters + sub;

  float cs[NP], sn[NP];
  if (p.norm) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (!known && lane == 0) index_error();
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      int a = 0, b = 0;
      const int pi = j + n * p.lanes;
      const bool turns = pi < p.npairs && pair_at<1, INTER>(p, pi, a, b);
      cs[n] = known ? 1.0f : NAN;  // a token without a position reads as NaN
      sn[n] = 0.0f;
      if (turns && known) load_turn<INTER>(p, pos, a, cs[n], sn[n]);
    }
  }
  const int64_t slot = p.slots ? load_index(p.slots, token, p.slot64) : -1;

  for (int it = 0; it < p.iters; ++it, head += per_warp) {
    const bool valid = head < heads;
    const bool is_q = head < p.hq, is_k = !is_q && head < p.hq + p.hk;
    const int h = is_q ? head : is_k ? head - p.hq : head - p.hq - p.hk;
    const T* x = is_q   ? static_cast<const T*>(p.q) + token * p.q_st + h * p.q_sh
                 : is_k ? static_cast<const T*>(p.k) + token * p.k_st + h * p.k_sh
                        : static_cast<const T*>(p.v) + token * p.v_st + h * p.v_sh;
    float xa[NP], xb[NP];
    float ss = 0.0f;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int pi = j + n * p.lanes;
      xa[n] = xb[n] = 0.0f;
      if (valid && pi < p.npairs) {
        int a, b;
        pair_at<1, INTER>(p, pi, a, b);
        xa[n] = to_f32<T>(x[a]);
        xb[n] = to_f32<T>(x[b]);
      }
      ss += xa[n] * xa[n] + xb[n] * xb[n];
    }
    if (p.norm) {
      ss = group_sum(ss, p.lanes);
      const float r = rsqrtf(ss / p.D + p.eps);
      if (valid && (is_q || is_k)) {
        const void* w = is_q ? p.qw : p.kw;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const int pi = j + n * p.lanes;
          if (pi < p.npairs) {
            int a, b;
            pair_at<1, INTER>(p, pi, a, b);
            float wa = 1.0f, wb = 1.0f;
            if (w) {
              wa = load_as(w, a, p.dtype_w);
              wb = load_as(w, b, p.dtype_w);
            }
            xa[n] = xa[n] * r * wa;
            xb[n] = xb[n] * r * wb;
            turn_pair(xa[n], xb[n], cs[n], sn[n], 1.0f);
          }
        }
      }
    }
    const bool cached = valid && !is_q && (!is_k || p.k_to_cache);
    float step = 0.0f;
    int64_t row = -1;
    if (p.slots) {  // uniform: every lane takes part in the row maximum
      float amax = 0.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n)
        amax = max_nan(amax, max_nan(fabsf(xa[n]), fabsf(xb[n])));
      for (int o = p.lanes >> 1; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      step = quantise_step(amax, p.cache.format);
      if (cached) row = slot_row(p.cache, slot, h);
    }
    if (cached) {
      if (row >= 0) {
        void* base = is_k ? p.cache.k : p.cache.v;
        if (p.cache.format >= OJX_KV_INT8 && j == 0) (is_k ? p.cache.k_scale : p.cache.v_scale)[row] = step;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const int pi = j + n * p.lanes;
          if (pi < p.npairs) {
            int a, b;
            pair_at<1, INTER>(p, pi, a, b);
            store_cached(base, row * p.D + a, p.cache.format, step, xa[n]);
            store_cached(base, row * p.D + b, p.cache.format, step, xb[n]);
          }
        }
      }
    } else if (valid) {
      T* out = is_q ? static_cast<T*>(p.q_out) + (token * p.hq + h) * p.D
                    : static_cast<T*>(p.k_out) + (token * p.hk + h) * p.D;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const int pi = j + n * p.lanes;
        if (pi < p.npairs) {
          int a, b;
          pair_at<1, INTER>(p, pi, a, b);
          out[a] = from_f32<T>(xa[n]);
          out[b] = from_f32<T>(xb[n]);
        }
      }
    }
  }
}

// Gradient rows.  Blocks [0, q_blocks) take query heads, the rest key heads; a warp walks
// tokens and all heads of its side, keeping its share of dw in registers; the block's
// sum goes to its own row of `partial`, so the result does not depend on timing.  (The
// same rows: 140 us.)
template <typename T, int NP, bool INTER>
__global__ void __launch_bounds__(256) qk_grad_kernel(const QkParams p) {
  extern __shared__ float sw[];  // [warps][D]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const bool is_q = blockIdx.x < p.q_blocks;
  const int block = is_q ? blockIdx.x : blockIdx.x - p.q_blocks;
  const int blocks = is_q ? p.q_blocks : gridDim.x - p.q_blocks;
  const int heads = is_q ? p.hq : p.hk;
  const T* xs = static_cast<const T*>(is_q ? p.q : p.k);
  const T* gs = static_cast<const T*>(is_q ? p.gq_data : p.gk_data);
  T* dxs = static_cast<T*>(is_q ? p.dq : p.dk);
  const int64_t x_st = is_q ? p.q_st : p.k_st, x_sh = is_q ? p.q_sh : p.k_sh;
  const int64_t g_st = is_q ? p.gq_st : p.gk_st, g_sh = is_q ? p.gq_sh : p.gk_sh;
  const void* w = is_q ? p.qw : p.kw;

  int at[NP][2];
  float wa[NP], wb[NP], da[NP], db[NP];
  bool on[NP], turns[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const int pi = j + n * p.lanes;
    on[n] = pi < p.npairs;
    at[n][0] = at[n][1] = 0;
    turns[n] = on[n] && pair_at<1, INTER>(p, pi, at[n][0], at[n][1]);
    wa[n] = wb[n] = 1.0f;
    da[n] = db[n] = 0.0f;
    if (w && on[n]) {
      wa[n] = load_as(w, at[n][0], p.dtype_w);
      wb[n] = load_as(w, at[n][1], p.dtype_w);
    }
  }
  const int row_groups = (heads + per_warp - 1) / per_warp;
  for (int64_t token = static_cast<int64_t>(block) * warps + warp; token < p.tokens;
       token += static_cast<int64_t>(blocks) * warps) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (!known && lane == 0) index_error();
    float cs[NP], sn[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      cs[n] = known ? 1.0f : NAN;
      sn[n] = 0.0f;
      if (turns[n] && known) load_turn<INTER>(p, pos, at[n][0], cs[n], sn[n]);
    }
    for (int rg = 0; rg < row_groups; ++rg) {
      const int h = rg * per_warp + sub;
      const bool valid = h < heads;
      const T* x = xs + token * x_st + h * x_sh;
      const T* g = gs + token * g_st + h * g_sh;
      float xa[NP], xb[NP], ga[NP], gb[NP];
      float ss = 0.0f, hx = 0.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        xa[n] = xb[n] = ga[n] = gb[n] = 0.0f;
        if (valid && on[n]) {
          xa[n] = to_f32<T>(x[at[n][0]]);
          xb[n] = to_f32<T>(x[at[n][1]]);
          ga[n] = to_f32<T>(g[at[n][0]]);
          gb[n] = to_f32<T>(g[at[n][1]]);
          turn_pair(ga[n], gb[n], cs[n], sn[n], -1.0f);
        }
        ss += xa[n] * xa[n] + xb[n] * xb[n];
        hx += ga[n] * wa[n] * xa[n] + gb[n] * wb[n] * xb[n];
      }
      for (int o = p.lanes >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        hx += __shfl_xor_sync(0xffffffffu, hx, o);
      }
      const float r = rsqrtf(ss / p.D + p.eps);
      const float back = r * r * hx / p.D;
      if (valid) {
        T* dx = dxs + (token * heads + h) * p.D;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          if (!on[n]) continue;
          const float oa = r * (ga[n] * wa[n] - xa[n] * back);
          const float ob = r * (gb[n] * wb[n] - xb[n] * back);
          da[n] += ga[n] * (xa[n] * r);
          db[n] += gb[n] * (xb[n] * r);
          dx[at[n][0]] = from_f32<T>(oa);
          dx[at[n][1]] = from_f32<T>(ob);
        }
      }
    }
  }
  // rows of the warp, then warps of the block, in a fixed order
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    for (int o = p.lanes; o < 32; o <<= 1) {
      da[n] += __shfl_xor_sync(0xffffffffu, da[n], o);
      db[n] += __shfl_xor_sync(0xffffffffu, db[n], o);
    }
    if (sub == 0 && on[n]) {
      sw[warp * p.D + at[n][0]] = da[n];
      sw[warp * p.D + at[n][1]] = db[n];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float s = 0.0f;
    for (int i = 0; i < warps; ++i) s += sw[i * p.D + d];
    p.partial[static_cast<int64_t>(blockIdx.x) * p.D + d] = s;
  }
}

// ── two float32 operations an instruction ──────────────────────────────────────────
__device__ __forceinline__ uint64_t f2_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t f2_swap(uint64_t v) {
  const float2 a = f2_split(v);
  return f2_pair(a.y, a.x);
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Eight elements as they lie in memory, and as four float32 pairs.
template <typename T>
struct Eight {
  uint4 v[8 * sizeof(T) / 16];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void pairs(uint64_t (&x)[4]) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = f2_pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[i] = f2_pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[i] = f2_pair(f.x, f.y);
      }
    }
  }
};
// Eight float32 values to eight elements of T: one store of 32 (float32: the widest there
// is) or 16 bytes.  (Stores of half a 32-byte sector each cost the L2 a transaction.)
template <typename T>
__device__ __forceinline__ void store_pairs(T* p, const uint64_t (&x)[4], bool wide) {
  if constexpr (sizeof(T) == 4) {
    const float2 a = f2_split(x[0]), b = f2_split(x[1]), c = f2_split(x[2]), d = f2_split(x[3]);
    if (wide) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x),
                   "f"(c.y), "f"(d.x), "f"(d.y)
                   : "memory");
    } else {
      reinterpret_cast<float4*>(p)[0] = make_float4(a.x, a.y, b.x, b.y);
      reinterpret_cast<float4*>(p)[1] = make_float4(c.x, c.y, d.x, d.y);
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = f2_split(x[i]);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void load_weight(const void* w, int at, int dtype, bool on, uint64_t (&x)[4]) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 1.0f;
  if (w && on) load_eight_as(w, at, dtype, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = f2_pair(v[2 * i], v[2 * i + 1]);
}

__device__ __forceinline__ bool table_aligned(const QkParams& p) {
  return ((p.rotary & 7) | (reinterpret_cast<uintptr_t>(p.table) & 15)) == 0;
}

// The turn of a chunk pair (a, b), in pairs of elements.  Halves: (c, s) of elements 2 i,
// 2 i + 1, the same for both chunks.  Interleaved: element pairs turn on themselves,
// (c, c) and (-s, s), each chunk with its own four.
template <bool INTER>
struct Turn {
  uint64_t c[INTER ? 8 : 4], s[INTER ? 8 : 4], n[INTER ? 1 : 4];  // (n: -s)
  // row: the position's cosines, its sines `half` further on.
  __device__ __forceinline__ void load(const float* table_row, int half, bool aligned, bool known, bool turns, int a) {
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = known ? 1.0f : NAN;  // a token without a position reads as NaN
      sn[e] = 0.0f;
    }
    if (turns && known) {
      const float* row = table_row + (INTER ? a / 2 : a);
      if (aligned) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 x = reinterpret_cast<const float4*>(row)[h], y = reinterpret_cast<const float4*>(row + half)[h];
          cs[4 * h] = x.x, cs[4 * h + 1] = x.y, cs[4 * h + 2] = x.z, cs[4 * h + 3] = x.w;
          sn[4 * h] = y.x, sn[4 * h + 1] = y.y, sn[4 * h + 2] = y.z, sn[4 * h + 3] = y.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          cs[e] = row[e];
          sn[e] = row[half + e];
        }
      }
    }
    if constexpr (INTER) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = f2_pair(cs[e], cs[e]);
        s[e] = f2_pair(-sn[e], sn[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = f2_pair(cs[2 * i], cs[2 * i + 1]);
        s[i] = f2_pair(sn[2 * i], sn[2 * i + 1]);
        n[i] = f2_pair(-sn[2 * i], -sn[2 * i + 1]);
      }
    }
  }
  // SIGN 1: by the angle, -1: back.
  template <int SIGN>
  __device__ __forceinline__ void apply(uint64_t (&a)[4], uint64_t (&b)[4]) const {
    [[maybe_unused]] const uint64_t minus = f2_pair(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (INTER) {
        const uint64_t sa = SIGN > 0 ? s[i] : f2_mul(s[i], minus), sb = SIGN > 0 ? s[4 + i] : f2_mul(s[4 + i], minus);
        a[i] = f2_fma(f2_swap(a[i]), sa, f2_mul(a[i], c[i]));
        b[i] = f2_fma(f2_swap(b[i]), sb, f2_mul(b[i], c[4 + i]));
      } else {
        const uint64_t u = a[i], v = b[i];
        a[i] = f2_fma(v, SIGN > 0 ? n[i] : s[i], f2_mul(u, c[i]));
        b[i] = f2_fma(u, SIGN > 0 ? s[i] : n[i], f2_mul(v, c[i]));
      }
    }
  }
};

__device__ __forceinline__ float f2_total(uint64_t v) {
  const float2 a = f2_split(v);
  return a.x + a.y;
}

// What is done with a row pair of chunks once it is in registers.  out: where the row goes
// if it is not cached; h: its head.
template <typename T, bool INTER>
__device__ __forceinline__ void norm_turn(const QkParams& p, const Turn<INTER>& turn, const uint64_t (&wa)[4], const uint64_t (&wb)[4],
                                          uint64_t (&xa)[4], uint64_t (&xb)[4]) {
  uint64_t ss = f2_mul(xa[0], xa[0]), tt = f2_mul(xb[0], xb[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    ss = f2_fma(xa[i], xa[i], ss);
    tt = f2_fma(xb[i], xb[i], tt);
  }
  const float r = rsqrtf(fmaf(group_sum(f2_total(f2_add(ss, tt)), p.lanes), p.inv_dim, p.eps));
  const uint64_t r2 = f2_pair(r, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    xa[i] = f2_mul(f2_mul(xa[i], r2), wa[i]);
    xb[i] = f2_mul(f2_mul(xb[i], r2), wb[i]);
  }
  turn.template apply<1>(xa, xb);
}
// x / step of two elements, correctly rounded, from inv = 1 / step rounded: an estimate
// x * inv and two corrections by its exact remainder (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990: the second correction
// of a quotient within one ulp rounds it correctly).  Needs steps far from under- and
// overflow.  The compiler's division took 40 % of the instructions of an append.
__device__ __forceinline__ uint64_t quotient2(uint64_t x, uint64_t minus_step, uint64_t inv) {
  uint64_t q = f2_mul(x, inv);
  q = f2_fma(f2_fma(q, minus_step, x), inv, q);
  return f2_fma(f2_fma(q, minus_step, x), inv, q);
}
// Eight elements of a row of this step as the cache's bytes.
__device__ __forceinline__ uint2 quantise_eight(const uint64_t (&x)[4], float step, int format) {
  uint32_t w[2] = {0, 0};
  if (step >= 8.67361738e-19f && step <= 1.15292150e18f) {  // 2^-60 .. 2^60
    const float inv = __frcp_rn(step);
    const uint64_t inv2 = f2_pair(inv, inv), minus = f2_pair(-step, -step);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 q = f2_split(quotient2(x[i], minus, inv2));
      uint32_t two;
      if (format == OJX_KV_INT8) {
        // rounding to whole by adding 1.5 * 2^23: the low byte is the two's complement
        const float u = fminf(fmaxf(q.x, -127.0f), 127.0f) + 12582912.0f, v = fminf(fmaxf(q.y, -127.0f), 127.0f) + 12582912.0f;
        two = __byte_perm(__float_as_uint(u), __float_as_uint(v), 0x0040);
      } else {
        two = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
      }
      w[i >> 1] |= (two & 0xffffu) << (16 * (i & 1));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = f2_split(x[i]);
      w[i >> 1] |= (quantise_one(v.x, step, format) | (static_cast<uint32_t>(quantise_one(v.y, step, format)) << 8)) << (16 * (i & 1));
    }
  }
  return make_uint2(w[0], w[1]);
}

// A row pair of chunks into the cache.
__device__ __forceinline__ void cache_row(const QkParams& p, int64_t slot, bool is_k, int h, bool valid, bool on, int j, int a, int b,
                                          const uint64_t (&xa)[4], const uint64_t (&xb)[4]) {
  void* base = is_k ? p.cache.k : p.cache.v;
  const int64_t row = valid ? slot_row(p.cache, slot, h) : -1;
  if (p.cache.format >= OJX_KV_INT8) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = f2_split(xa[i]), v = f2_split(xb[i]);
      amax = max_nan(amax, max_nan(max_nan(fabsf(u.x), fabsf(u.y)), max_nan(fabsf(v.x), fabsf(v.y))));
    }
    for (int o = p.lanes >> 1; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float step = quantise_step(amax, p.cache.format);
    if (row < 0 || !on) return;
    if (j == 0) (is_k ? p.cache.k_scale : p.cache.v_scale)[row] = step;
    uint8_t* dst = static_cast<uint8_t*>(base) + row * p.D;
    *reinterpret_cast<uint2*>(dst + a) = quantise_eight(xa, step, p.cache.format);
    *reinterpret_cast<uint2*>(dst + b) = quantise_eight(xb, step, p.cache.format);
  } else if (row >= 0 && on) {
    if (p.cache.format == OJX_KV_BF16) {
      store_pairs<__nv_bfloat16>(static_cast<__nv_bfloat16*>(base) + row * p.D + a, xa, false);
      store_pairs<__nv_bfloat16>(static_cast<__nv_bfloat16*>(base) + row * p.D + b, xb, false);
    } else {
      store_pairs<__half>(static_cast<__half*>(base) + row * p.D + a, xa, false);
      store_pairs<__half>(static_cast<__half*>(base) + row * p.D + b, xb, false);
    }
  }
}

// Forward rows in 16-byte chunks.  A group is 32 / lanes heads of one side (queries, keys,
// values) of a token; a warp runs p.iters groups of one token with the next two groups'
// loads in flight: at 16 warps an SM that covers HBM's latency.  One group at a time took
// 116 us for 16384 tokens of 40 bf16 heads of 128.  A few tokens (8: 3.3 us) are one
// dependent round of loads.
template <typename T, bool INTER, bool NORM>
__global__ void __launch_bounds__(256, 2) qk_rows_fast_kernel(const QkParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  const int64_t token = item / p.blocks_per_token;
  if (token >= p.tokens) return;  // whole warp
  const int first = static_cast<int>(item - token * p.blocks_per_token) * p.iters;
  const int end = min(first + p.iters, p.gq + p.gk + p.gv);
  const bool on = j < p.npairs;
  int a = 0, b = 0;
  const bool turns = on && pair_at<8, INTER>(p, j, a, b);

  auto fetch = [&](int g, Eight<T>& xa, Eight<T>& xb) {
    const bool is_q = g < p.gq, is_k = !is_q && g < p.gq + p.gk;
    const int h = (g - (is_q ? 0 : is_k ? p.gq : p.gq + p.gk)) * per_warp + sub;
    const int heads = is_q ? p.hq : is_k ? p.hk : p.hv;
    xa.clear();
    xb.clear();
    if (g < end && on && h < heads) {
      const T* x = is_q   ? static_cast<const T*>(p.q) + token * p.q_st + h * p.q_sh
                   : is_k ? static_cast<const T*>(p.k) + token * p.k_st + h * p.k_sh
                          : static_cast<const T*>(p.v) + token * p.v_st + h * p.v_sh;
      xa.load(x + a);
      xb.load(x + b);
    }
  };
  Eight<T> a0, b0, a1, b1;
  fetch(first, a0, b0);
  fetch(first + 1, a1, b1);

  Turn<INTER> turn;
  uint64_t wa[4], wb[4];
  if (NORM) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (!known && lane == 0) index_error();
    turn.load(p.table + (known ? pos : 0) * p.rotary, p.half, table_aligned(p), known, turns, a);
  }
  const int64_t slot = p.slots ? load_index(p.slots, token, p.slot64) : -1;
  const bool wide_q = (reinterpret_cast<uintptr_t>(p.q_out) & 31) == 0, wide_k = (reinterpret_cast<uintptr_t>(p.k_out) & 31) == 0;
  int side = -1;  // whose weights wa and wb are
#pragma unroll 2
  for (int g = first; g < end; ++g) {
    const bool is_q = g < p.gq, is_k = !is_q && g < p.gq + p.gk;  // uniform
    const int h = (g - (is_q ? 0 : is_k ? p.gq : p.gq + p.gk)) * per_warp + sub;
    const bool valid = h < (is_q ? p.hq : is_k ? p.hk : p.hv);
    uint64_t xa[4], xb[4];
    a0.pairs(xa);
    b0.pairs(xb);
    a0 = a1;
    b0 = b1;
    fetch(g + 2, a1, b1);
    if (NORM && (is_q || is_k)) {
      if (side != (is_q ? 0 : 1)) {
        side = is_q ? 0 : 1;
        load_weight(is_q ? p.qw : p.kw, a, p.dtype_w, on, wa);
        load_weight(is_q ? p.qw : p.kw, b, p.dtype_w, on, wb);
      }
      norm_turn<T, INTER>(p, turn, wa, wb, xa, xb);
    }
    if (is_q || (is_k && !p.k_to_cache)) {
      if (valid && on) {
        T* out = is_q ? static_cast<T*>(p.q_out) + (token * p.hq + h) * p.D : static_cast<T*>(p.k_out) + (token * p.hk + h) * p.D;
        store_pairs<T>(out + a, xa, is_q ? wide_q : wide_k);
        store_pairs<T>(out + b, xb, is_q ? wide_q : wide_k);
      }
    } else {
      cache_row(p, slot, is_k, h, valid, on, j, a, b, xa, xb);
    }
  }
}

// A block's sum of dw: rows of a warp, then warps, in a fixed order.  sw: [warps][D].
__device__ __forceinline__ void grad_weight_sums(const QkParams& p, float* sw, bool store, int a, int b, uint64_t (&da)[4],
                                                 uint64_t (&db)[4]) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int o = p.lanes; o < 32; o <<= 1) {
      da[i] = f2_add(da[i], __shfl_xor_sync(0xffffffffu, da[i], o));
      db[i] = f2_add(db[i], __shfl_xor_sync(0xffffffffu, db[i], o));
    }
    if (store) {
      *reinterpret_cast<float2*>(&sw[warp * p.D + a + 2 * i]) = f2_split(da[i]);
      *reinterpret_cast<float2*>(&sw[warp * p.D + b + 2 * i]) = f2_split(db[i]);
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float s = 0.0f;
    for (int i = 0; i < warps; ++i) s += sw[i * p.D + d];
    p.partial[static_cast<int64_t>(blockIdx.x) * p.D + d] = s;
  }
}

template <typename T, bool INTER>
__device__ __forceinline__ void grad_group(const QkParams& p, bool store, T* dx, int a, int b, bool wide, const Turn<INTER>& turn,
                                           const uint64_t (&wa)[4], const uint64_t (&wb)[4], const uint64_t (&xa)[4],
                                           const uint64_t (&xb)[4], uint64_t (&ga)[4], uint64_t (&gb)[4], uint64_t (&da)[4],
                                           uint64_t (&db)[4]) {
  turn.template apply<-1>(ga, gb);
  uint64_t ss = 0, hx = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ss = f2_fma(xa[i], xa[i], ss);
    ss = f2_fma(xb[i], xb[i], ss);
    hx = f2_fma(f2_mul(ga[i], wa[i]), xa[i], hx);
    hx = f2_fma(f2_mul(gb[i], wb[i]), xb[i], hx);
  }
  float s1 = f2_total(ss), s2 = f2_total(hx);
  for (int o = p.lanes >> 1; o > 0; o >>= 1) {
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    s2 += __shfl_xor_sync(0xffffffffu, s2, o);
  }
  const float r = rsqrtf(fmaf(s1, p.inv_dim, p.eps));
  const float back = -(r * r * s2 * p.inv_dim);
  const uint64_t r2 = f2_pair(r, r), back2 = f2_pair(back, back);
  if (store) {
    uint64_t oa[4], ob[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      oa[i] = f2_mul(f2_fma(xa[i], back2, f2_mul(ga[i], wa[i])), r2);
      ob[i] = f2_mul(f2_fma(xb[i], back2, f2_mul(gb[i], wb[i])), r2);
      da[i] = f2_fma(ga[i], f2_mul(xa[i], r2), da[i]);
      db[i] = f2_fma(gb[i], f2_mul(xb[i], r2), db[i]);
    }
    store_pairs<T>(dx + a, oa, wide);
    store_pairs<T>(dx + b, ob, wide);
  }
}

// Gradient rows in 16-byte chunks, the next group's two loads in flight; otherwise as
// qk_grad_kernel.
template <typename T, bool INTER>
__global__ void __launch_bounds__(256, 2) qk_grad_fast_kernel(const QkParams p) {
  extern __shared__ float sw[];  // [warps][D]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const bool is_q = blockIdx.x < p.q_blocks;
  const int block = is_q ? blockIdx.x : blockIdx.x - p.q_blocks;
  const int blocks = is_q ? p.q_blocks : gridDim.x - p.q_blocks;
  const int heads = is_q ? p.hq : p.hk, groups = is_q ? p.gq : p.gk;
  const T* xs = static_cast<const T*>(is_q ? p.q : p.k);
  const T* gs = static_cast<const T*>(is_q ? p.gq_data : p.gk_data);
  T* dxs = static_cast<T*>(is_q ? p.dq : p.dk);
  const int64_t x_st = is_q ? p.q_st : p.k_st, x_sh = is_q ? p.q_sh : p.k_sh;
  const int64_t g_st = is_q ? p.gq_st : p.gk_st, g_sh = is_q ? p.gq_sh : p.gk_sh;
  const bool wide = (reinterpret_cast<uintptr_t>(dxs) & 31) == 0;
  const bool on = j < p.npairs;
  int a = 0, b = 0;
  const bool turns = on && pair_at<8, INTER>(p, j, a, b);
  uint64_t wa[4], wb[4], da[4], db[4];
  load_weight(is_q ? p.qw : p.kw, a, p.dtype_w, on, wa);
  load_weight(is_q ? p.qw : p.kw, b, p.dtype_w, on, wb);
#pragma unroll
  for (int i = 0; i < 4; ++i) da[i] = db[i] = 0;

  const int64_t stride = static_cast<int64_t>(blocks) * warps;
  int64_t token = static_cast<int64_t>(block) * warps + warp;
  int64_t next_token = token;  // of the loads in flight
  int next_group = 0;
  Eight<T> ra, rb, sa, sb;
  auto fetch = [&]() {
    const int h = next_group * per_warp + sub;
    ra.clear(), rb.clear(), sa.clear(), sb.clear();
    if (next_token < p.tokens && on && h < heads) {
      const T* x = xs + next_token * x_st + h * x_sh;
      const T* g = gs + next_token * g_st + h * g_sh;
      ra.load(x + a);
      rb.load(x + b);
      sa.load(g + a);
      sb.load(g + b);
    }
    if (++next_group == groups) next_group = 0, next_token += stride;
  };
  fetch();
  Turn<INTER> turn;
  for (; token < p.tokens; token += stride) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (!known && lane == 0) index_error();
    turn.load(p.table + (known ? pos : 0) * p.rotary, p.half, table_aligned(p), known, turns, a);
    for (int rg = 0; rg < groups; ++rg) {
      const int h = rg * per_warp + sub;
      uint64_t xa[4], xb[4], ga[4], gb[4];
      ra.pairs(xa);
      rb.pairs(xb);
      sa.pairs(ga);
      sb.pairs(gb);
      fetch();
      grad_group<T, INTER>(p, h < heads && on, dxs + (token * heads + h) * p.D, a, b, wide, turn, wa, wb, xa, xb, ga, gb, da, db);
    }
  }
  grad_weight_sums(p, sw, sub == 0 && on, a, b, da, db);
}

// ── rows streamed through shared memory ─────────────────────────────────────────
// With many tokens whose heads lie side by side, a warp takes an equal run of all groups
// and keeps a ring of them in flight: one bulk copy a group (its rows are one piece of
// memory) into the warp's own ring, and with a token's first group the position's row of
// the table.  A group is two rows a lane (float32: one): what is done once a group, the
// wait, the next copy and the addresses, then weighs half as much, and instructions are
// what bounds these kernels once the loads are ahead.  16384 tokens of 40 heads of 128, bf16:
// forward 56 us (6.0 TB/s), gradient 96 us (5.2 TB/s); 8192 tokens of 48 heads, 16 of them to
// int8 pages, 51 us; append of 50021 tokens of 4 heads, f32 to int8, 76 us (3.4 TB/s: the
// quotients).
// (Two float32 rows, with the ring of three that then fits, appended 50021 tokens in 92 us,
// one with a ring of four in 77.)
template <typename T>
inline constexpr int qk_rows_per_lane = sizeof(T) == 4 ? 1 : 2;
constexpr int QK_RING = 4, QK_GRAD_RING = 2;

struct StreamAt {  // the group that is issued, or used, next
  int u, token, g;
  __device__ __forceinline__ void begin(int first, int groups) {
    u = first;
    token = first / groups;
    g = first - token * groups;
  }
  __device__ __forceinline__ bool next(int groups) {  // true: a new token
    ++u;
    if (++g < groups) return false;
    g = 0;
    ++token;
    return true;
  }
};

// Both weights as float32 in shared memory: [2][D].
__device__ __forceinline__ void stage_weights(const QkParams& p, float* sw) {
  for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
    const void* w = i < p.D ? p.qw : p.kw;
    sw[i] = w ? load_as(w, i < p.D ? i : i - p.D, p.dtype_w) : 1.0f;
  }
}
__device__ __forceinline__ void staged_weight(const float* w, bool on, uint64_t (&x)[4]) {
  if (!on) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const ulonglong2 v = reinterpret_cast<const ulonglong2*>(w)[h];
    x[2 * h] = v.x;
    x[2 * h + 1] = v.y;
  }
}

template <typename T, bool INTER, bool NORM>
__global__ void __launch_bounds__(256, 2) qk_rows_stream_kernel(const QkParams p, int slot_bytes, uint64_t budget) {
  constexpr int RPL = qk_rows_per_lane<T>;
  extern __shared__ __align__(128) uint8_t smem[];  // [8 warps][QK_RING][group | table row], then both weights
  __shared__ __align__(8) uint64_t bars[8 * QK_RING];
  __shared__ int s_known[8 * QK_RING], s_abort;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const int groups = p.gq + p.gk + p.gv;
  const int group_bytes = RPL * per_warp * p.D * static_cast<int>(sizeof(T));
  const uint32_t bar = smem_u32(&bars[warp * QK_RING]);
  uint8_t* ring = smem + warp * QK_RING * slot_bytes;
  const float* sw = reinterpret_cast<const float*>(smem + 8 * QK_RING * slot_bytes);
  if (lane < QK_RING) mbar_init(bar + 8 * lane, 1);
  if (threadIdx.x == 0) s_abort = 0;
  if (NORM) stage_weights(p, reinterpret_cast<float*>(smem + 8 * QK_RING * slot_bytes));
  fence_mbar_init();
  __syncthreads();

  const long long total = p.tokens * groups, warps = static_cast<long long>(gridDim.x) * 8, w = static_cast<long long>(blockIdx.x) * 8 + warp;
  const int first = static_cast<int>(total * w / warps), end = static_cast<int>(total * (w + 1) / warps);
  StreamAt in, at;
  in.begin(first, groups);
  at = in;
  // (positions are read a token ahead of the copy that needs them)
  int64_t pos = NORM && first < end ? load_index(p.positions, in.token, p.pos64) : 0;
  int in_slot = 0;
  auto issue = [&]() {
    if (in.u >= end) return;
    if (lane == 0) {
      const bool is_q = in.g < p.gq, is_k = !is_q && in.g < p.gq + p.gk;
      const int h = (in.g - (is_q ? 0 : is_k ? p.gq : p.gq + p.gk)) * (RPL * per_warp);
      const int rows = min(RPL * per_warp, (is_q ? p.hq : is_k ? p.hk : p.hv) - h);
      const bool fresh = NORM && (in.g == 0 || in.u == first), known = pos >= 0 && pos < p.table_rows;
      const T* x = static_cast<const T*>(is_q ? p.q : is_k ? p.k : p.v) + in.token * (is_q ? p.q_st : is_k ? p.k_st : p.v_st);
      const uint32_t dst = smem_u32(ring + in_slot * slot_bytes), full = bar + 8 * in_slot;
      const uint32_t bytes = rows * p.D * sizeof(T), row = fresh && known ? p.rotary * 4 : 0;
      mbar_arrive_expect_tx(full, bytes + row);
      bulk_load_g2s(dst, x + h * p.D, bytes, full);
      if (fresh) {
        if (!known) index_error();
        s_known[warp * QK_RING + in_slot] = known;
        if (row) bulk_load_g2s(dst + group_bytes, p.table + pos * p.rotary, row, full);
      }
    }
    if (in.next(groups) && NORM && in.u < end) pos = load_index(p.positions, in.token, p.pos64);
    in_slot = in_slot + 1 == QK_RING ? 0 : in_slot + 1;
  };
#pragma unroll 1
  for (int i = 0; i < QK_RING; ++i) issue();
  __syncwarp();  // lane 0's s_known of these groups (later ones: the loop's)

  const bool on = j < p.npairs;
  int a = 0, b = 0;
  const bool turns = on && pair_at<8, INTER>(p, j, a, b);
  const bool wide_q = (reinterpret_cast<uintptr_t>(p.q_out) & 31) == 0, wide_k = (reinterpret_cast<uintptr_t>(p.k_out) & 31) == 0;
  Turn<INTER> turn;
  uint64_t wa[4] = {0, 0, 0, 0}, wb[4] = {0, 0, 0, 0};
  int slot_at = 0;
  uint32_t phase = 0;
  int64_t slot = -1;
  while (at.u < end) {
    const bool is_q = at.g < p.gq, is_k = !is_q && at.g < p.gq + p.gk, fresh = at.g == 0 || at.u == first;
    const int h0 = (at.g - (is_q ? 0 : is_k ? p.gq : p.gq + p.gk)) * (RPL * per_warp) + sub, heads = is_q ? p.hq : is_k ? p.hk : p.hv;
    if (fresh && p.slots) slot = load_index(p.slots, at.token, p.slot64);
    if (NORM && (fresh || at.g == p.gq)) {  // the side changes
      staged_weight(sw + (is_q ? a : p.D + a), on, wa);
      staged_weight(sw + (is_q ? b : p.D + b), on, wb);
    }
    if (!__all_sync(0xffffffffu, mbar_wait(bar + 8 * slot_at, phase, budget, &s_abort))) break;
    const uint8_t* src = ring + slot_at * slot_bytes;
    if (NORM && fresh)
      turn.load(reinterpret_cast<const float*>(src + group_bytes), p.half, (p.rotary & 7) == 0, s_known[warp * QK_RING + slot_at] != 0, turns, a);
    Eight<T> ra[RPL], rb[RPL];
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      ra[r].clear();
      rb[r].clear();
      if (h0 + r * per_warp < heads && on) {
        const T* x = reinterpret_cast<const T*>(src) + (sub + r * per_warp) * p.D;
        ra[r].load(x + a);
        rb[r].load(x + b);
      }
    }
    uint64_t xa[RPL][4], xb[RPL][4];
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      ra[r].pairs(xa[r]);
      rb[r].pairs(xb[r]);
    }
    __syncwarp();  // the slot is read
    issue();
    if (is_q || (is_k && !p.k_to_cache)) {
      T* out = static_cast<T*>(is_q ? p.q_out : p.k_out) + static_cast<int64_t>(at.token) * (heads * p.D) + h0 * p.D;
#pragma unroll
      for (int r = 0; r < RPL; ++r) {
        if (NORM) norm_turn<T, INTER>(p, turn, wa, wb, xa[r], xb[r]);
        if (h0 + r * per_warp < heads && on) {
          store_pairs<T>(out + r * per_warp * p.D + a, xa[r], is_q ? wide_q : wide_k);
          store_pairs<T>(out + r * per_warp * p.D + b, xb[r], is_q ? wide_q : wide_k);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < RPL; ++r) {
        if (NORM && is_k) norm_turn<T, INTER>(p, turn, wa, wb, xa[r], xb[r]);
        cache_row(p, slot, is_k, h0 + r * per_warp, h0 + r * per_warp < heads, on, j, a, b, xa[r], xb[r]);
      }
    }
    at.next(groups);
    if (++slot_at == QK_RING) slot_at = 0, phase ^= 1;
  }
  // (after a wait that ran out: let the copies in flight land before the block may exit)
  for (; at.u < in.u; at.next(groups)) {
    mbar_wait_drain(bar + 8 * slot_at, phase, budget);
    if (++slot_at == QK_RING) slot_at = 0, phase ^= 1;
  }
}

template <typename T, bool INTER>
__global__ void __launch_bounds__(256, 2) qk_grad_stream_kernel(const QkParams p, int slot_bytes, uint64_t budget) {
  constexpr int RPL = qk_rows_per_lane<T>, RING = QK_GRAD_RING;
  extern __shared__ __align__(128) uint8_t smem[];  // [8 warps][RING][rows | gradients | table row]; at the end [8][D] sums
  __shared__ __align__(8) uint64_t bars[8 * RING];
  __shared__ int s_known[8 * RING], s_abort;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const bool is_q = blockIdx.x < p.q_blocks;
  const int block = is_q ? blockIdx.x : blockIdx.x - p.q_blocks;
  const int blocks = is_q ? p.q_blocks : gridDim.x - p.q_blocks;
  const int heads = is_q ? p.hq : p.hk, groups = is_q ? p.gq : p.gk;
  const T* xs = static_cast<const T*>(is_q ? p.q : p.k);
  const T* gs = static_cast<const T*>(is_q ? p.gq_data : p.gk_data);
  T* dxs = static_cast<T*>(is_q ? p.dq : p.dk);
  const int64_t x_st = is_q ? p.q_st : p.k_st, g_st = is_q ? p.gq_st : p.gk_st;
  const int group_bytes = RPL * per_warp * p.D * static_cast<int>(sizeof(T));
  const uint32_t bar = smem_u32(&bars[warp * RING]);
  uint8_t* ring = smem + warp * RING * slot_bytes;
  if (lane < RING) mbar_init(bar + 8 * lane, 1);
  if (threadIdx.x == 0) s_abort = 0;
  fence_mbar_init();
  __syncthreads();

  const long long total = p.tokens * groups, warps = static_cast<long long>(blocks) * 8, w = static_cast<long long>(block) * 8 + warp;
  const int first = static_cast<int>(total * w / warps), end = static_cast<int>(total * (w + 1) / warps);
  StreamAt in, at;
  in.begin(first, groups);
  at = in;
  int64_t pos = first < end ? load_index(p.positions, in.token, p.pos64) : 0;
  int in_slot = 0;
  auto issue = [&]() {
    if (in.u >= end) return;
    if (lane == 0) {
      const int h = in.g * (RPL * per_warp), rows = min(RPL * per_warp, heads - h);
      const bool fresh = in.g == 0 || in.u == first, known = pos >= 0 && pos < p.table_rows;
      const uint32_t dst = smem_u32(ring + in_slot * slot_bytes), full = bar + 8 * in_slot;
      const uint32_t bytes = rows * p.D * sizeof(T), row = fresh && known ? p.rotary * 4 : 0;
      mbar_arrive_expect_tx(full, 2 * bytes + row);
      bulk_load_g2s(dst, xs + in.token * x_st + h * p.D, bytes, full);
      bulk_load_g2s(dst + group_bytes, gs + in.token * g_st + h * p.D, bytes, full);
      if (fresh) {
        if (!known) index_error();
        s_known[warp * RING + in_slot] = known;
        if (row) bulk_load_g2s(dst + 2 * group_bytes, p.table + pos * p.rotary, row, full);
      }
    }
    if (in.next(groups) && in.u < end) pos = load_index(p.positions, in.token, p.pos64);
    in_slot = in_slot + 1 == RING ? 0 : in_slot + 1;
  };
#pragma unroll 1
  for (int i = 0; i < RING; ++i) issue();
  __syncwarp();  // lane 0's s_known of these groups (later ones: the loop's)

  const bool wide = (reinterpret_cast<uintptr_t>(dxs) & 31) == 0;
  const bool on = j < p.npairs;
  int a = 0, b = 0;
  const bool turns = on && pair_at<8, INTER>(p, j, a, b);
  uint64_t wa[4], wb[4], da[4], db[4];
  load_weight(is_q ? p.qw : p.kw, a, p.dtype_w, on, wa);
  load_weight(is_q ? p.qw : p.kw, b, p.dtype_w, on, wb);
#pragma unroll
  for (int i = 0; i < 4; ++i) da[i] = db[i] = 0;
  Turn<INTER> turn;
  int slot_at = 0;
  uint32_t phase = 0;
  while (at.u < end) {
    const int h0 = at.g * (RPL * per_warp) + sub;
    if (!__all_sync(0xffffffffu, mbar_wait(bar + 8 * slot_at, phase, budget, &s_abort))) break;
    const uint8_t* src = ring + slot_at * slot_bytes;
    if (at.g == 0 || at.u == first)
      turn.load(reinterpret_cast<const float*>(src + 2 * group_bytes), p.half, (p.rotary & 7) == 0, s_known[warp * RING + slot_at] != 0, turns, a);
    T* dx = dxs + static_cast<int64_t>(at.token) * (heads * p.D) + h0 * p.D;
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      const bool mine = h0 + r * per_warp < heads && on;
      Eight<T> ra, rb, ga_, gb_;
      ra.clear(), rb.clear(), ga_.clear(), gb_.clear();
      if (mine) {
        const T* x = reinterpret_cast<const T*>(src) + (sub + r * per_warp) * p.D;
        const T* g = reinterpret_cast<const T*>(src + group_bytes) + (sub + r * per_warp) * p.D;
        ra.load(x + a);
        rb.load(x + b);
        ga_.load(g + a);
        gb_.load(g + b);
      }
      uint64_t xa[4], xb[4], ga[4], gb[4];
      ra.pairs(xa);
      rb.pairs(xb);
      ga_.pairs(ga);
      gb_.pairs(gb);
      if (r == RPL - 1) {
        __syncwarp();  // the slot is read
        issue();
      }
      grad_group<T, INTER>(p, mine, dx + r * per_warp * p.D, a, b, wide, turn, wa, wb, xa, xb, ga, gb, da, db);
    }
    at.next(groups);
    if (++slot_at == RING) slot_at = 0, phase ^= 1;
  }
  for (; at.u < in.u; at.next(groups)) {
    mbar_wait_drain(bar + 8 * slot_at, phase, budget);
    if (++slot_at == RING) slot_at = 0, phase ^= 1;
  }
  __syncthreads();
  grad_weight_sums(p, reinterpret_cast<float*>(smem), sub == 0 && on, a, b, da, db);
}

__device__ __forceinline__ void store_as(void* p, int64_t at, int dtype, float v) {
  if (dtype == OJX_F32) static_cast<float*>(p)[at] = v;
  else if (dtype == OJX_BF16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[at] = __float2half_rn(v);
}

// dw of one side: its blocks' partial sums, in 32 interleaved runs of blocks joined in
// order.  grid (ceil(D / 32), 2), 32 x 32 threads.  Bound by latency: 3.2 us for 296 blocks.
__global__ void __launch_bounds__(1024) qk_grad_weight_kernel(const float* partial, int q_blocks, int blocks, int D, void* dqw, void* dkw,
                                                              int dtype) {
  __shared__ float s[32][33];
  const int d = blockIdx.x * 32 + threadIdx.x;
  void* out = blockIdx.y == 0 ? dqw : dkw;
  const int lo = blockIdx.y == 0 ? 0 : q_blocks, hi = blockIdx.y == 0 ? q_blocks : blocks;
  float v = 0.0f;
  if (d < D) {
#pragma unroll 4
    for (int b = lo + threadIdx.y; b < hi; b += 32) v += partial[static_cast<int64_t>(b) * D + d];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && d < D && out) {
#pragma unroll
    for (int i = 1; i < 32; ++i) v += s[i][threadIdx.x];
    store_as(out, d, dtype, v);
  }
}

// Rows of the cache at `slots` as dense [n][heads][D] keys and values; a skipped slot
// gives zeros.  A thread takes eight elements of a row's key and value, and of the rows
// two, so four loads are in flight.  50021 tokens of 4 heads, int8 to f32: 46 us (5.6 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const ojx_kv_cache c, const void* slots, int slot64, int64_t n,
                                                      T* k_out, T* v_out) {
  const int cpr = c.head_dim / 8, per_block = 256 / cpr;  // rows that a block takes at a time
  const int r0 = threadIdx.x / cpr, at = (threadIdx.x - r0 * cpr) * 8;
  if (r0 >= per_block) return;
  const int64_t rows = n * c.kv_heads;
  const bool wide = ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 31) == 0;
  int64_t r[2], row[2];
  uint4 k[2], v[2];
  float ks[2], vs[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    r[u] = (static_cast<int64_t>(blockIdx.x) * 2 + u) * per_block + r0;
    row[u] = -1;
    if (r[u] < rows) {
      const int64_t token = r[u] / c.kv_heads;
      row[u] = slot_row(c, load_index(slots, token, slot64), static_cast<int>(r[u] - token * c.kv_heads));
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    k[u] = v[u] = make_uint4(0, 0, 0, 0);
    ks[u] = vs[u] = 0.0f;
    if (row[u] < 0) continue;
    const int64_t src = row[u] * c.head_dim + at;
    if (c.format >= OJX_KV_INT8) {
      const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(c.k) + src);
      const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(c.v) + src);
      k[u].x = a.x, k[u].y = a.y, v[u].x = b.x, v[u].y = b.y;
      ks[u] = c.k_scale[row[u]];
      vs[u] = c.v_scale[row[u]];
    } else {
      k[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.k) + src);
      v[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.v) + src);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (r[u] >= rows) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 w = h ? v[u] : k[u];
      const float step = h ? vs[u] : ks[u];
      uint64_t x[4];
      if (c.format == OJX_KV_BF16) {
        Eight<__nv_bfloat16> e;
        e.v[0] = w;
        e.pairs(x);
      } else if (c.format == OJX_KV_F16) {
        Eight<__half> e;
        e.v[0] = w;
        e.pairs(x);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t two = (i < 2 ? w.x : w.y) >> (16 * (i & 1));
          x[i] = f2_pair(dequantise_one(static_cast<uint8_t>(two), step, c.format), dequantise_one(static_cast<uint8_t>(two >> 8), step, c.format));
        }
        if (row[u] < 0) x[0] = x[1] = x[2] = x[3] = 0;
      }
      store_pairs<T>((h ? v_out : k_out) + r[u] * c.head_dim + at, x, wide);
    }
  }
}

// Moves the rows of the accepted nodes path[b][0..count[b]] of the drafts at context +
// node to context + 0, 1, ...  One block per (sequence, head); a thread owns a 16-byte
// column of the rows and moves them in path order.  A node's index is at least its
// place in the path, so a row is read before a later row is written over it.  64 sequences,
// 5 accepted of 48: 8.2 us, the latency of a chain of moves.
__global__ void __launch_bounds__(128) kv_keep_path_kernel(const ojx_kv_cache c, const int32_t* page_table, int width,
                                                           const int32_t* contexts, const int32_t* path,
                                                           const int32_t* count, int tokens) {
  const int b = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
  const int es = c.format >= OJX_KV_INT8 ? 1 : 2;
  const int cols = c.head_dim * es / 16;
  const int scales = c.format >= OJX_KV_INT8 ? 2 : 0;
  const int t = threadIdx.x;
  if (t >= 2 * cols + scales) return;
  const int n = min(count[b], tokens - 1);
  const int64_t ctx = contexts[b];
  auto row_of = [&](int64_t key) -> int64_t {
    const int64_t pg = key / c.page_size;
    if (key < 0 || pg >= width) return -1;
    const int64_t id = page_table[static_cast<int64_t>(b) * width + pg];
    if (id < 0 || id >= c.num_pages) return -1;
    return (id * c.kv_heads + h) * c.page_size + key % c.page_size;
  };
  int before = -1;
  for (int i = 0; i <= n; ++i) {
    const int node = path[static_cast<int64_t>(b) * tokens + i];
    const bool ordered = node > before && node < tokens;
    const int64_t src = ordered ? row_of(ctx + node) : -1, dst = row_of(ctx + i);
    if (src < 0 || dst < 0) {
      if (t == 0) index_error();
      return;
    }
    before = node;
    if (src == dst) continue;
    if (t < 2 * cols) {
      uint4* base = static_cast<uint4*>(t < cols ? c.k : c.v);
      const int col = t % cols;
      base[dst * cols + col] = base[src * cols + col];
    } else {
      float* base = t == 2 * cols ? c.k_scale : c.v_scale;
      base[dst] = base[src];
    }
  }
}

}  // namespace ojx
