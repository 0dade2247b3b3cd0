// verify.cuh — verification of drafted tokens against the target's probabilities, from
// given random numbers.
//
// Drafts form a tree: node 0 is the root (known), node i > 0 carries token x_i and was
// drafted after parents[i] < i; row n of `target` (p) and `draft` (q) are the
// distributions of the token that follows node n.  Nodes are tried in index order, each
// when its parent is the node reached.  With r = p_n, W = 1 on reaching n:
//   accept x_i when u_i q(x_i) W < r(x_i)  (then n = i);
//   else r <- max(r - W q, 0), W <- the mass of r, and the next child is tried.
// Without draft rows a draft is a certainty (q = 1 at x_i): a rejected token's r becomes 0
// and W falls by it.  The next token is drawn from what is left of r by u_0: the first v
// with cumulated weight > floor(u_0 * total).  Weights are whole numbers, floor(r 2^38),
// so sums are exact in any order: masses and tokens do not depend on how the row is
// split over threads.
//
// A cluster of up to eight CTAs serves one sequence, each an equal part of the row; they exchange
// their sums through distributed shared memory.  The walk needs no row pass but for the
// mass between siblings (draft rows given): a warp finds the children of the node reached
// by ballot, so its steps are the nodes that are tried.  One pass finds the total; the warp
// whose share holds the token sums strips of it, one a lane, and then reads one strip.
// Bound by the latency of its dependent steps for few sequences (4 chains of 6 drafts over
// 32000 tokens with draft rows: 12 us), and for many by that and the one (two) rows read per
// sequence (64 trees of 48 nodes over 131072 tokens: 27 us, of which 34 MB are 5).
#pragma once
#include <cooperative_groups.h>
#include "qk_cache.cuh"

namespace ojx {

constexpr int VD_CLUSTER = 8;  // CTAs of a sequence, at most
constexpr int VD_THREADS = 512;
constexpr int VD_WARPS = VD_THREADS / 32;
constexpr int VD_MAX_TOKENS = 1024;

struct VerifyParams {
  const void *target, *draft;
  int64_t t_sb, t_st, d_sb, d_st;  // strides of sequences and nodes, in elements
  const int32_t *tokens, *parents;
  const float* uniforms;
  int32_t *path, *count, *next;
  int T;
  int64_t V;
};

// A probability as it counts: 0 for NaN and below, at most 1.
template <typename T>
__device__ __forceinline__ float vd_prob(const T* p, int64_t i) {
  return fminf(fmaxf(to_f32<T>(p[i]), 0.0f), 1.0f);
}
// floor(r * 2^38) for r in [0, 1]: the significand, 15 bits up, and down by the exponent.
// (The conversion instructions run at a sixteenth of the integer ones' rate.)
__device__ __forceinline__ unsigned long long vd_units(float r) {
  const uint32_t bits = __float_as_uint(r);
  const unsigned long long m = static_cast<unsigned long long>((bits & 0x7fffffu) | 0x800000u) << 15;
  return bits < 0x2c000000u ? 0ull : m >> (127u - (bits >> 23));  // below 2^-39: nothing
}
// Elements of a row that one warp of the cluster takes: whole vectors.
__host__ __device__ constexpr int64_t vd_per_warp(int64_t V, int cluster) {
  return ((V + cluster * VD_WARPS - 1) / (cluster * VD_WARPS) + 3) / 4 * 4;
}
// Four neighbouring probabilities (elements from `n` on: 0).
template <typename T>
__device__ __forceinline__ void vd_load4(const T* p, int n, bool vec, float (&r)[4]) {
  if (vec && n >= 4) {
    T e[4];
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
    else *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = vd_prob<T>(e, i);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = i < n ? vd_prob<T>(p, i) : 0.0f;
  }
}
// r after the rejections with masses ws[0 .. k) at one node
__device__ __forceinline__ float vd_left(float r, float q, const float* ws, int k) {
  for (int i = 0; i < k; ++i) r = fmaxf(__fsub_rn(r, __fmul_rn(ws[i], q)), 0.0f);
  return r;
}

template <typename T>
__global__ void __launch_bounds__(VD_THREADS, 2)
    verify_drafts_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ uint32_t s_gone[];  // bit per token of this CTA's share: rejected (no draft rows)
  __shared__ int s_parent[VD_MAX_TOKENS], s_token[VD_MAX_TOKENS];
  __shared__ float s_u[VD_MAX_TOKENS], s_p[VD_MAX_TOKENS], s_q[VD_MAX_TOKENS];
  __shared__ float s_ws[VD_MAX_TOKENS];
  __shared__ unsigned long long s_sum[2][VD_CLUSTER], s_warp[VD_WARPS];
  __shared__ int s_state[4];  // node reached, rejections at it, next node to try, needs a mass
  __shared__ int s_gone_list[VD_MAX_TOKENS];
  __shared__ uint8_t s_again[VD_MAX_TOKENS];  // an earlier sibling has the same token

  const int rank = static_cast<int>(cluster.block_rank());
  const int ctas = static_cast<int>(cluster.num_blocks());
  const int64_t b = blockIdx.x / ctas;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* target = static_cast<const T*>(p.target) + b * p.t_sb;
  const T* draft = p.draft ? static_cast<const T*>(p.draft) + b * p.d_sb : nullptr;

  // Each CTA holds every node's own probabilities, so all take the same decisions.
  for (int i = tid; i < p.T; i += VD_THREADS) {
    int par = p.parents[b * p.T + i];
    const int tok = p.tokens[b * p.T + i];
    float pp = 0.0f, qq = 1.0f;
    if (i > 0) {
      const bool absent = tok < 0;  // padding of a smaller tree
      if (!absent && (tok >= p.V || par < 0 || par >= i)) {
        if (rank == 0) index_error();
        par = -1;
      } else if (absent) {
        par = -1;
      } else {
        pp = vd_prob<T>(target + par * p.t_st, tok);
        if (draft) qq = vd_prob<T>(draft + par * p.d_st, tok);
      }
    }
    s_parent[i] = i > 0 ? par : -1;
    s_token[i] = tok;
    s_u[i] = p.uniforms[b * p.T + i];
    s_p[i] = pp;
    s_q[i] = qq;
  }
  if (tid == 0) {
    s_state[0] = 0;
    s_state[1] = 0;
    s_state[2] = 1;
    s_ws[0] = 1.0f;
    if (rank == 0) p.path[b * p.T] = 0;
  }
  if (!draft) {
    __syncthreads();
    for (int i = tid; i < p.T; i += VD_THREADS) {
      bool again = false;
      for (int e = 1; e < i; ++e) again |= s_parent[e] == s_parent[i] && s_token[e] == s_token[i];
      s_again[i] = again;
    }
  }
  cluster.sync();  // every CTA runs before its shared memory is written from another

  // this CTA's share of a row, and this warp's share of that
  const int64_t per_warp = vd_per_warp(p.V, ctas);
  const int64_t lo = min(p.V, (static_cast<int64_t>(rank) * VD_WARPS + warp) * per_warp);
  const int64_t hi = min(p.V, lo + per_warp);
  int taken = 0, turn = 0;

  auto vectors = [](const T* row) { return (reinterpret_cast<uintptr_t>(row) & (4 * sizeof(T) - 1)) == 0; };
  // Weights of elements v .. v + 3 (those below `n` of them), each in w if asked for.
  auto weight4 = [&](const T* pr, const T* qr, int64_t v, int n, int k, bool gone, bool vec, unsigned long long* w = nullptr) {
    float r[4], q[4];
    vd_load4<T>(pr + v, n, vec, r);
    if (qr && k) {
      vd_load4<T>(qr + v, n, vec, q);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = vd_left(r[i], q[i], s_ws, k);
    }
    if (gone) {
      const int64_t at = v - static_cast<int64_t>(rank) * VD_WARPS * per_warp;  // a multiple of four
      const uint32_t bits = s_gone[at >> 5] >> (at & 31);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((bits >> i) & 1) r[i] = 0.0f;
    }
    unsigned long long sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long x = vd_units(r[i]);
      if (w) w[i] = x;
      sum += x;
    }
    return sum;
  };

  // Total of floor(r 2^38) over the row of `node` after k rejections; fills s_warp and
  // s_sum[which] (this CTA's warps, all CTAs).  Called by every thread of the cluster.
  auto total_of = [&](int node, int k, bool gone, int which) {
    const T* pr = target + node * p.t_st;
    const T* qr = draft ? draft + node * p.d_st : nullptr;
    unsigned long long sum = 0;
    const bool vec = vectors(pr) && (!qr || vectors(qr));
    const int n = static_cast<int>(hi - lo);
#pragma unroll 4
    for (int v = lane * 4; v < n; v += 128) sum += weight4(pr, qr, lo + v, n - v, k, gone, vec);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    if (tid < ctas) {
      unsigned long long all = 0;
      for (int i = 0; i < VD_WARPS; ++i) all += s_warp[i];
      cluster.map_shared_rank(&s_sum[which][0], tid)[rank] = all;
    }
    cluster.sync();
    unsigned long long all = 0;
    for (int i = 0; i < ctas; ++i) all += s_sum[which][i];
    return all;
  };

  while (true) {
    if (warp == 0) {  // (every lane follows the walk; lane 0 writes)
      int node = s_state[0], k = s_state[1], i = s_state[2], want = 0;
      int accepted = taken;
      float mass = s_ws[draft ? k : 0];
      __syncwarp();
      while (true) {
        // the next node from i on whose parent is the one reached
        int next = p.T;
        for (int base = i & ~31; base < p.T; base += 32) {
          const int c = base + lane;
          const unsigned hit = __ballot_sync(0xffffffffu, c >= i && c < p.T && s_parent[c] == node);
          if (hit) {
            next = base + __ffs(hit) - 1;
            break;
          }
        }
        i = next;
        if (i >= p.T) break;
        if (draft && mass < 0.0f) {  // the mass after k rejections is not known yet
          want = 1;
          break;
        }
        float r = s_p[i];
        if (draft) r = vd_left(r, s_q[i], s_ws, k);
        else if (s_again[i]) r = 0.0f;
        if (__fmul_rn(s_u[i], __fmul_rn(s_q[i], mass)) < r) {
          node = i;
          k = 0;
          mass = 1.0f;
          ++accepted;
          if (lane == 0) {
            s_ws[0] = 1.0f;
            if (rank == 0) p.path[b * p.T + accepted] = i;
          }
        } else if (draft) {
          ++k;
          mass = -1.0f;
          if (lane == 0) s_ws[k] = -1.0f;
        } else {
          mass = fmaxf(__fsub_rn(mass, r), 0.0f);
          if (lane == 0) {
            s_gone_list[k] = s_token[i];
            s_ws[0] = mass;
          }
          ++k;
        }
        ++i;
        __syncwarp();
      }
      if (lane == 0) {
        s_state[0] = node;
        s_state[1] = k;
        s_state[2] = i;
        s_state[3] = want;
      }
      taken = accepted;
    }
    __syncthreads();
    if (!s_state[3]) break;
    const unsigned long long m = total_of(s_state[0], s_state[1], false, turn);
    turn ^= 1;  // the other CTAs may still read the sums of this turn
    if (tid == 0) s_ws[s_state[1]] = static_cast<float>(static_cast<double>(m) / 274877906944.0);
    __syncthreads();
  }

  const int node = s_state[0];
  int k = s_state[1];
  bool gone = !draft && k > 0;
  const int64_t base = static_cast<int64_t>(rank) * VD_WARPS * per_warp;
  if (gone) {
    const int words = static_cast<int>((VD_WARPS * per_warp + 31) / 32);
    for (int i = tid; i < words; i += VD_THREADS) s_gone[i] = 0;
    __syncthreads();
    for (int i = tid; i < k; i += VD_THREADS) {
      const int64_t at = s_gone_list[i] - base;
      if (at >= 0 && at < VD_WARPS * per_warp) atomicOr(&s_gone[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
  }
  unsigned long long total = total_of(node, k, gone, turn);
  if (total == 0) {  // nothing left by rounding: the node's own row
    turn ^= 1;
    k = 0;
    gone = false;
    __syncthreads();
    total = total_of(node, 0, false, turn);
  }
  if (rank == 0) {
    if (tid == 0) {
      p.count[b] = taken;
      if (total == 0) p.next[b] = -1;
      s_state[2] = taken;
    }
    __syncthreads();
    for (int i = s_state[2] + 1 + tid; i < p.T; i += VD_THREADS) p.path[b * p.T + i] = -1;
  }
  const float u0 = s_u[0];
  const long long u24 = min(max(__float2ll_rd(u0 * 16777216.0f), 0ll), (1ll << 24) - 1);
  const unsigned long long goal = static_cast<unsigned long long>(u24) * (total >> 24) +
                                  ((static_cast<unsigned long long>(u24) * (total & 0xffffffull)) >> 24);
  unsigned long long before = 0;
  for (int i = 0; i < rank; ++i) before += s_sum[turn][i];
  for (int i = 0; i < warp; ++i) before += s_warp[i];
  if (total > 0 && before <= goal && goal < before + s_warp[warp]) {  // one warp of the cluster
    const T* pr = target + node * p.t_st;
    const T* qr = draft ? draft + node * p.d_st : nullptr;
    const bool vec = vectors(pr) && (!qr || vectors(qr));
    const int n = static_cast<int>(hi - lo);
    const int strip = ((n + 31) / 32 + 3) / 4 * 4;
    const int s0 = min(n, lane * strip), s1 = min(n, s0 + strip);
    unsigned long long mine = 0;
#pragma unroll 4
    for (int v = s0; v < s1; v += 4) mine += weight4(pr, qr, lo + v, s1 - v, k, gone, vec);
    unsigned long long run = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + run > goal);  // (not empty: goal lies in this warp's share)
    const int src = __ffs(hit) - 1;
    before += __shfl_sync(0xffffffffu, run - mine, src);
    const int t0 = min(n, src * strip), t1 = min(n, t0 + strip);
    for (int v0 = t0; v0 < t1; v0 += 128) {
      const int v = v0 + 4 * lane;
      unsigned long long w[4] = {0, 0, 0, 0};
      unsigned long long four = 0;
      if (v < t1) four = weight4(pr, qr, lo + v, t1 - v, k, gone, vec, w);
      unsigned long long up_to = four;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, up_to, o);
        if (lane >= o) up_to += up;
      }
      const unsigned in = __ballot_sync(0xffffffffu, before + up_to > goal);
      if (in) {
        if (lane == __ffs(in) - 1) {
          unsigned long long at = before + up_to - four;
          int i = 0;
          while (i < 3 && at + w[i] <= goal) at += w[i++];
          p.next[b] = static_cast<int32_t>(lo + v + i);
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, up_to, 31);
    }
  }
  cluster.sync();  // no CTA leaves while another may still write its shared sums
}

}  // namespace ojx
