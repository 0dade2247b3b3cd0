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
// A lane holds CH elements of both halves of a pair, so the rotation needs no exchange
// between lanes, and 32 / lanes-per-row rows share a warp.
#pragma once
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

// CH consecutive elements as fp32.  CH = 8 reads 16-byte vectors (p 16-byte aligned).
template <typename T, int CH>
__device__ __forceinline__ void load_chunk(const T* p, float (&v)[CH]) {
  if constexpr (CH == 8) {
    constexpr int NV = 8 * sizeof(T) / 16;
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = to_f32<T>(p[i]);
  }
}
template <typename T, int CH>
__device__ __forceinline__ void store_chunk(T* p, const float (&v)[CH]) {
  if constexpr (CH == 8) {
    constexpr int NV = 8 * sizeof(T) / 16;
    uint4 raw[NV];
    T* e = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i) p[i] = from_f32<T>(v[i]);
  }
}
// The same from memory whose type is only known at run time (weights).
template <int CH>
__device__ __forceinline__ void load_chunk_as(const void* p, int64_t at, int dtype, float (&v)[CH]) {
  if (dtype == OJX_F32) load_chunk<float, CH>(static_cast<const float*>(p) + at, v);
  else if (dtype == OJX_BF16) load_chunk<__nv_bfloat16, CH>(static_cast<const __nv_bfloat16*>(p) + at, v);
  else load_chunk<__half, CH>(static_cast<const __half*>(p) + at, v);
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
  int dtype_w, pos64, slot64, k_to_cache;
  float eps;
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
  const void *gq, *gk;
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

// Cosines and sines of one pair chunk: cs[e], sn[e] belong to pair e of the chunk pair.
// (INTER, CH = 8: pairs 0-3 lie in the first chunk, 4-7 in the second.)
template <int CH, bool INTER>
__device__ __forceinline__ void load_turn(const QkParams& p, int64_t pos, int a, float (&cs)[CH], float (&sn)[CH]) {
  const float* row = p.table + pos * p.rotary;
  const int first = INTER ? a / 2 : a;
#pragma unroll
  for (int e = 0; e < CH; ++e) {
    cs[e] = row[first + e];
    sn[e] = row[p.half + first + e];
  }
}

// Turn a chunk pair by the angle (sign = 1) or back (sign = -1).
template <int CH, bool INTER>
__device__ __forceinline__ void turn_pair(float (&xa)[CH], float (&xb)[CH], const float (&cs)[CH],
                                          const float (&sn)[CH], float sign) {
  if constexpr (INTER && CH > 1) {
#pragma unroll
    for (int e = 0; e < CH / 2; ++e) {
      float u = xa[2 * e], v = xa[2 * e + 1], s = sign * sn[e];
      xa[2 * e] = u * cs[e] - v * s;
      xa[2 * e + 1] = u * s + v * cs[e];
      u = xb[2 * e], v = xb[2 * e + 1], s = sign * sn[CH / 2 + e];
      xb[2 * e] = u * cs[CH / 2 + e] - v * s;
      xb[2 * e + 1] = u * s + v * cs[CH / 2 + e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      const float u = xa[e], v = xb[e], s = sign * sn[e];
      xa[e] = u * cs[e] - v * s;
      xb[e] = u * s + v * cs[e];
    }
  }
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

template <int CH>
__device__ __forceinline__ void store_cached(void* base, int64_t at, int format, float step, const float (&v)[CH]) {
  if (format == OJX_KV_BF16) {
    store_chunk<__nv_bfloat16, CH>(static_cast<__nv_bfloat16*>(base) + at, v);
  } else if (format == OJX_KV_F16) {
    store_chunk<__half, CH>(static_cast<__half*>(base) + at, v);
  } else {
    uint8_t q[CH];
#pragma unroll
    for (int e = 0; e < CH; ++e) q[e] = quantise_one(v[e], step, format);
    uint8_t* dst = static_cast<uint8_t*>(base) + at;
    if constexpr (CH == 8) {
      uint2 w;
      w.x = q[0] | (q[1] << 8) | (q[2] << 16) | (static_cast<uint32_t>(q[3]) << 24);
      w.y = q[4] | (q[5] << 8) | (q[6] << 16) | (static_cast<uint32_t>(q[7]) << 24);
      *reinterpret_cast<uint2*>(dst) = w;
    } else {
#pragma unroll
      for (int e = 0; e < CH; ++e) dst[e] = q[e];
    }
  }
}

// Forward rows: query and key heads are normed and rotated (p.norm) and stored densely
// or, keys with k_to_cache and all value heads, into the cache.  A warp takes one token
// and p.iters row groups of it, so the token's cosines are loaded once for its heads.
template <typename T, int CH, int NP, bool INTER>
__global__ void __launch_bounds__(256) qk_rows_kernel(const QkParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  const int64_t token = item / p.blocks_per_token;
  if (token >= p.tokens) return;  // whole warp
  const int heads = p.hq + p.hk + p.hv;
  int head = static_cast<int>(item % p.blocks_per_token) * per_warp * p.iters + sub;

  float cs[NP][CH], sn[NP][CH];
  if (p.norm) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (!known && lane == 0) index_error();
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      int a = 0, b = 0;
      const int pi = j + n * p.lanes;
      const bool turns = pi < p.npairs && pair_at<CH, INTER>(p, pi, a, b);
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        cs[n][e] = known ? 1.0f : NAN;  // a token without a position reads as NaN
        sn[n][e] = 0.0f;
      }
      if (turns && known) load_turn<CH, INTER>(p, pos, a, cs[n], sn[n]);
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
    float xa[NP][CH], xb[NP][CH];
    float ss = 0.0f;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int pi = j + n * p.lanes;
#pragma unroll
      for (int e = 0; e < CH; ++e) xa[n][e] = xb[n][e] = 0.0f;
      if (valid && pi < p.npairs) {
        int a, b;
        pair_at<CH, INTER>(p, pi, a, b);
        load_chunk<T, CH>(x + a, xa[n]);
        load_chunk<T, CH>(x + b, xb[n]);
      }
#pragma unroll
      for (int e = 0; e < CH; ++e) ss += xa[n][e] * xa[n][e] + xb[n][e] * xb[n][e];
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
            pair_at<CH, INTER>(p, pi, a, b);
            float wa[CH], wb[CH];
            if (w) {
              load_chunk_as<CH>(w, a, p.dtype_w, wa);
              load_chunk_as<CH>(w, b, p.dtype_w, wb);
            }
#pragma unroll
            for (int e = 0; e < CH; ++e) {
              xa[n][e] = xa[n][e] * r * (w ? wa[e] : 1.0f);
              xb[n][e] = xb[n][e] * r * (w ? wb[e] : 1.0f);
            }
            turn_pair<CH, INTER>(xa[n], xb[n], cs[n], sn[n], 1.0f);
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
#pragma unroll
        for (int e = 0; e < CH; ++e) amax = max_nan(amax, max_nan(fabsf(xa[n][e]), fabsf(xb[n][e])));
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
            pair_at<CH, INTER>(p, pi, a, b);
            store_cached<CH>(base, row * p.D + a, p.cache.format, step, xa[n]);
            store_cached<CH>(base, row * p.D + b, p.cache.format, step, xb[n]);
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
          pair_at<CH, INTER>(p, pi, a, b);
          store_chunk<T, CH>(out + a, xa[n]);
          store_chunk<T, CH>(out + b, xb[n]);
        }
      }
    }
  }
}

// Gradient rows.  Blocks [0, q_blocks) take query heads, the rest key heads; a warp walks
// tokens and all heads of its side, keeping its share of dw in registers; the block's
// sum goes to its own row of `partial`, so the result does not depend on timing.
template <typename T, int CH, int NP, bool INTER>
__global__ void __launch_bounds__(256) qk_grad_kernel(const QkParams p) {
  extern __shared__ float sw[];  // [warps][D]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int sub = lane / p.lanes, j = lane % p.lanes, per_warp = 32 / p.lanes;
  const bool is_q = blockIdx.x < p.q_blocks;
  const int block = is_q ? blockIdx.x : blockIdx.x - p.q_blocks;
  const int blocks = is_q ? p.q_blocks : gridDim.x - p.q_blocks;
  const int heads = is_q ? p.hq : p.hk;
  const T* xs = static_cast<const T*>(is_q ? p.q : p.k);
  const T* gs = static_cast<const T*>(is_q ? p.gq : p.gk);
  T* dxs = static_cast<T*>(is_q ? p.dq : p.dk);
  const int64_t x_st = is_q ? p.q_st : p.k_st, x_sh = is_q ? p.q_sh : p.k_sh;
  const int64_t g_st = is_q ? p.gq_st : p.gk_st, g_sh = is_q ? p.gq_sh : p.gk_sh;
  const void* w = is_q ? p.qw : p.kw;

  int at[NP][2];
  float wa[NP][CH], wb[NP][CH], da[NP][CH], db[NP][CH];
  bool on[NP], turns[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const int pi = j + n * p.lanes;
    on[n] = pi < p.npairs;
    at[n][0] = at[n][1] = 0;
    turns[n] = on[n] && pair_at<CH, INTER>(p, pi, at[n][0], at[n][1]);
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      wa[n][e] = wb[n][e] = 1.0f;
      da[n][e] = db[n][e] = 0.0f;
    }
    if (w && on[n]) {
      load_chunk_as<CH>(w, at[n][0], p.dtype_w, wa[n]);
      load_chunk_as<CH>(w, at[n][1], p.dtype_w, wb[n]);
    }
  }
  const int row_groups = (heads + per_warp - 1) / per_warp;
  for (int64_t token = static_cast<int64_t>(block) * warps + warp; token < p.tokens;
       token += static_cast<int64_t>(blocks) * warps) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (!known && lane == 0) index_error();
    float cs[NP][CH], sn[NP][CH];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        cs[n][e] = known ? 1.0f : NAN;
        sn[n][e] = 0.0f;
      }
      if (turns[n] && known) load_turn<CH, INTER>(p, pos, at[n][0], cs[n], sn[n]);
    }
    for (int rg = 0; rg < row_groups; ++rg) {
      const int h = rg * per_warp + sub;
      const bool valid = h < heads;
      const T* x = xs + token * x_st + h * x_sh;
      const T* g = gs + token * g_st + h * g_sh;
      float xa[NP][CH], xb[NP][CH], ga[NP][CH], gb[NP][CH];
      float ss = 0.0f, hx = 0.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
#pragma unroll
        for (int e = 0; e < CH; ++e) xa[n][e] = xb[n][e] = ga[n][e] = gb[n][e] = 0.0f;
        if (valid && on[n]) {
          load_chunk<T, CH>(x + at[n][0], xa[n]);
          load_chunk<T, CH>(x + at[n][1], xb[n]);
          load_chunk<T, CH>(g + at[n][0], ga[n]);
          load_chunk<T, CH>(g + at[n][1], gb[n]);
          turn_pair<CH, INTER>(ga[n], gb[n], cs[n], sn[n], -1.0f);
        }
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          ss += xa[n][e] * xa[n][e] + xb[n][e] * xb[n][e];
          hx += ga[n][e] * wa[n][e] * xa[n][e] + gb[n][e] * wb[n][e] * xb[n][e];
        }
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
          float oa[CH], ob[CH];
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            oa[e] = r * (ga[n][e] * wa[n][e] - xa[n][e] * back);
            ob[e] = r * (gb[n][e] * wb[n][e] - xb[n][e] * back);
            da[n][e] += ga[n][e] * (xa[n][e] * r);
            db[n][e] += gb[n][e] * (xb[n][e] * r);
          }
          store_chunk<T, CH>(dx + at[n][0], oa);
          store_chunk<T, CH>(dx + at[n][1], ob);
        }
      }
    }
  }
  // rows of the warp, then warps of the block, in a fixed order
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      for (int o = p.lanes; o < 32; o <<= 1) {
        da[n][e] += __shfl_xor_sync(0xffffffffu, da[n][e], o);
        db[n][e] += __shfl_xor_sync(0xffffffffu, db[n][e], o);
      }
      if (sub == 0 && on[n]) {
        sw[warp * p.D + at[n][0] + e] = da[n][e];
        sw[warp * p.D + at[n][1] + e] = db[n][e];
      }
    }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float s = 0.0f;
    for (int i = 0; i < warps; ++i) s += sw[i * p.D + d];
    p.partial[static_cast<int64_t>(blockIdx.x) * p.D + d] = s;
  }
}

__device__ __forceinline__ void store_as(void* p, int64_t at, int dtype, float v) {
  if (dtype == OJX_F32) static_cast<float*>(p)[at] = v;
  else if (dtype == OJX_BF16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[at] = __float2half_rn(v);
}

// dw of one side: its blocks' partial sums in block order.  grid (ceil(D / 32), 2),
// 32 x 8 threads: eight interleaved runs of blocks, joined in order.
__global__ void __launch_bounds__(256) qk_grad_weight_kernel(const float* partial, int q_blocks, int blocks, int D,
                                                             void* dqw, void* dkw, int dtype) {
  __shared__ float s[8][33];
  const int d = blockIdx.x * 32 + threadIdx.x;
  void* out = blockIdx.y == 0 ? dqw : dkw;
  const int lo = blockIdx.y == 0 ? 0 : q_blocks, hi = blockIdx.y == 0 ? q_blocks : blocks;
  float v = 0.0f;
  if (d < D)
    for (int b = lo + threadIdx.y; b < hi; b += 8) v += partial[static_cast<int64_t>(b) * D + d];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && d < D && out) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += s[i][threadIdx.x];
    store_as(out, d, dtype, v);
  }
}

// Rows of the cache at `slots` as dense [n][heads][D] keys and values; a skipped slot
// gives zeros.  One thread reads eight elements of one row.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const ojx_kv_cache c, const void* slots, int slot64, int64_t n,
                                                      T* k_out, T* v_out) {
  const int cpr = c.head_dim / 8;
  const int64_t per = n * c.kv_heads * cpr;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= 2 * per) return;
  const bool is_v = i >= per;
  const int64_t r = (is_v ? i - per : i) / cpr;
  const int at = static_cast<int>((is_v ? i - per : i) % cpr) * 8;
  const int64_t row = slot_row(c, load_index(slots, r / c.kv_heads, slot64), static_cast<int>(r % c.kv_heads));
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (row >= 0) {
    const void* base = is_v ? c.v : c.k;
    const int64_t src = row * c.head_dim + at;
    if (c.format == OJX_KV_BF16) {
      load_chunk<__nv_bfloat16, 8>(static_cast<const __nv_bfloat16*>(base) + src, x);
    } else if (c.format == OJX_KV_F16) {
      load_chunk<__half, 8>(static_cast<const __half*>(base) + src, x);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + src);
      const float step = (is_v ? c.v_scale : c.k_scale)[row];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = dequantise_one(static_cast<uint8_t>((e < 4 ? w.x : w.y) >> (8 * (e & 3))), step, c.format);
    }
  }
  store_chunk<T, 8>((is_v ? v_out : k_out) + r * c.head_dim + at, x);
}

// Moves the rows of the accepted nodes path[b][0..count[b]] of the drafts at context +
// node to context + 0, 1, ...  One block per (sequence, head); a thread owns a 16-byte
// column of the rows and moves them in path order.  A node's index is at least its
// place in the path, so a row is read before a later row is written over it.
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
