// serving.cu — the serving operators' kernels and their C-ABI (include/ojx.h): argument
// checks, launch shapes and workspaces.  A translation unit of its own, with its own
// device error word, so that it compiles beside the GEMM kernels.
#include <algorithm>
#include <mutex>
#include <type_traits>
#include "tmap.h"
#include "qk_cache.cuh"
#include "tree_attention.cuh"
#include "tree_attention_tc.cuh"
#include "verify.cuh"

namespace ojx {

// Devices on which a serving kernel has ever been launched or recorded by a capture: their
// error word is read at every poll from then on, for a kernel may still be running, or be
// replayed by a graph, long after the last call.
constexpr int MAX_DEVICES = 128;
static std::atomic<bool> g_serving_used[MAX_DEVICES];
static int device_slot() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev >= 0 && dev < MAX_DEVICES ? dev : 0;
}

// Fetched and cleared in one step, so that no bit that is set meanwhile is lost.
__device__ unsigned int g_taken_error = 0;
__global__ void take_serving_error_kernel() { g_taken_error = atomicExch(&g_dev_error, 0u); }

int serving_error_address(const unsigned int** address) {
  *address = nullptr;
  if (!g_serving_used[device_slot()].load(std::memory_order_relaxed)) return OJX_OK;
  void* p = nullptr;
  int st = cuda_status(cudaGetSymbolAddress(&p, g_dev_error), "serving error word");
  *address = static_cast<const unsigned int*>(p);
  return st;
}

int read_and_clear_serving_error(unsigned int* word) {
  int st = OJX_OK;
  take_serving_error_kernel<<<1, 1>>>();
  if ((st = cuda_status(cudaGetLastError(), "take serving error word"))) return st;
  return cuda_status(cudaMemcpyFromSymbol(word, g_taken_error, sizeof(unsigned int)), "take serving error word");
}

static int launched(const char* what) {
  g_launches.fetch_add(1);
  g_serving_used[device_slot()].store(true, std::memory_order_relaxed);
  return cuda_status(cudaGetLastError(), what);
}

// Two kernels that hand over through their stream's workspace are launched one right after
// the other: a call of another thread on the same stream must neither come between them nor
// replace (grow) the workspace before the second one has it.
static std::mutex& pair_mutex() {
  static std::mutex mu;
  return mu;
}

static bool known_dtype(int dt) { return dt == OJX_F32 || dt == OJX_BF16 || dt == OJX_F16; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int check_cache(const char* who, const ojx_kv_cache* c) {
  if (!c) return set_error(OJX_ERR_INVALID, "%s: cache is NULL", who);
  if (c->format < OJX_KV_BF16 || c->format > OJX_KV_FP8)
    return set_error(OJX_ERR_INVALID, "%s: unknown cache format %d", who, c->format);
  if (c->num_pages < 1 || c->page_size < 1 || c->kv_heads < 1)
    return set_error(OJX_ERR_INVALID, "%s: a cache has at least one page, row and head", who);
  if (c->num_pages > INT32_MAX) return set_error(OJX_ERR_INVALID, "%s: too many pages", who);
  if (c->head_dim < 16 || c->head_dim > 512 || c->head_dim % 16)
    return set_error(OJX_ERR_INVALID, "%s: head_dim %d is not a multiple of 16 up to 512", who, c->head_dim);
  if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v))
    return set_error(OJX_ERR_INVALID, "%s: cache pages must be 16-byte aligned", who);
  if (c->format >= OJX_KV_INT8 && (!c->k_scale || !c->v_scale))
    return set_error(OJX_ERR_INVALID, "%s: an 8-bit cache needs its steps", who);
  return OJX_OK;
}

// Whether rows can be read as 16-byte vectors.
static bool vector_rows(const ojx_rows& r, int es) {
  return !r.data || (aligned16(r.data) && (r.stride_t * es) % 16 == 0 && (r.stride_h * es) % 16 == 0);
}
// Whether every chunk of eight elements lies wholly inside or outside the turning part,
// and pairs of chunks cover a row.
static bool vector_pairs(int D, int rotary, bool inter) {
  if (D % 16 || D > 512) return false;
  return inter ? rotary % 16 == 0 : (rotary / 2) % 8 == 0 && (D - rotary) % 16 == 0;
}
static int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

template <typename F>
static int for_dtype(int dtype, F f) {
  if (dtype == OJX_F32) return f(float{});
  if (dtype == OJX_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

// Whether a token's heads lie side by side, so that a group of rows is one copy.
static bool side_by_side(int64_t stride_h, int D, int heads) { return heads <= 1 || stride_h == D; }

static int launch_rows(QkParams& p, int dtype, bool vec, bool inter, cudaStream_t s) {
  if (p.tokens == 0) return OJX_OK;
  const int CH = vec ? 8 : 1;
  p.npairs = p.D / (2 * CH);
  p.lanes = std::min(32, pow2_at_least(p.npairs));
  const int per_warp = 32 / p.lanes, heads = p.hq + p.hk + p.hv;
  p.gq = (p.hq + per_warp - 1) / per_warp;
  p.gk = (p.hk + per_warp - 1) / per_warp;
  p.gv = (p.hv + per_warp - 1) / per_warp;
  const int groups = vec ? p.gq + p.gk + p.gv : (heads + per_warp - 1) / per_warp;
  // One warp runs all heads of a token, so that the token's cosines are read once, unless
  // that leaves SMs without work: then its heads are split over more warps.
  const int64_t want = 16ll * current_props().sm_count;
  int split = 1;
  while (split < groups && p.tokens * split < want) split *= 2;
  split = std::min(split, groups);
  p.iters = (groups + split - 1) / split;
  p.blocks_per_token = (groups + p.iters - 1) / p.iters;
  // Streaming pays once each warp's ring fills several times; fewer tokens leave the loads to
  // prefetching in registers.  The rule counts tokens, so that is true of many heads: with few,
  // a warp has few groups (1537 tokens of 8 float32 heads: two), and only 40 heads of 128 were
  // timed both ways.  Streamed / prefetched, those heads in bf16: 400 tokens 4.8 / 4.4 us (with int8 caching 8.7 / 9.5), 800 tokens 6.3 / 8.7 (10.2 /
  // 13.2), 2400 tokens 11.9 / 17.6 (18.7 / 25.5).
  const int sms = current_props().sm_count;
  const bool table_ok = !p.norm || (aligned16(p.table) && p.rotary % 4 == 0);
  if (vec && table_ok && p.tokens >= 4ll * sms && side_by_side(p.q_sh, p.D, p.hq) && side_by_side(p.k_sh, p.D, p.hk) &&
      side_by_side(p.v_sh, p.D, p.hv)) {
    const int heads_each = (dtype == OJX_F32 ? 1 : 2) * per_warp;
    p.gq = (p.hq + heads_each - 1) / heads_each;
    p.gk = (p.hk + heads_each - 1) / heads_each;
    p.gv = (p.hv + heads_each - 1) / heads_each;
    if (p.tokens * (p.gq + p.gk + p.gv) > INT32_MAX) return set_error(OJX_ERR_INVALID, "too many rows for one call");
    const int slot = heads_each * p.D * dtype_size(dtype) + (p.norm ? p.rotary * 4 : 0);
    const int smem = 8 * QK_RING * slot + (p.norm ? 2 * p.D * 4 : 0);
    return for_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      auto go = [&](auto kern) {
        int st = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
        if (st) return st;
        kern<<<2 * sms, 256, smem, s>>>(p, slot, g_wait_budget.load());
        return launched("qk_rows_stream launch");
      };
      if (!p.norm) return go(qk_rows_stream_kernel<T, false, false>);
      return inter ? go(qk_rows_stream_kernel<T, true, true>) : go(qk_rows_stream_kernel<T, false, true>);
    });
  }
  const int64_t warps = p.tokens * p.blocks_per_token;
  const int64_t grid = (warps + 7) / 8;
  if (grid > INT32_MAX) return set_error(OJX_ERR_INVALID, "too many rows for one call");
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const unsigned gr = static_cast<unsigned>(grid);
    if (vec && !p.norm) qk_rows_fast_kernel<T, false, false><<<gr, 256, 0, s>>>(p);
    else if (vec && !inter) qk_rows_fast_kernel<T, false, true><<<gr, 256, 0, s>>>(p);
    else if (vec) qk_rows_fast_kernel<T, true, true><<<gr, 256, 0, s>>>(p);
    // (rows of up to 128 elements hold two pairs a lane, not eight: 4096 tokens of 40 heads of
    // 100, bf16, 68 us against 162; their gradient 140 against 307)
    else if (p.npairs <= 64 && !inter) qk_rows_kernel<T, 2, false><<<gr, 256, 0, s>>>(p);
    else if (p.npairs <= 64) qk_rows_kernel<T, 2, true><<<gr, 256, 0, s>>>(p);
    else if (!inter) qk_rows_kernel<T, 8, false><<<gr, 256, 0, s>>>(p);
    else qk_rows_kernel<T, 8, true><<<gr, 256, 0, s>>>(p);
    return launched("qk_rows launch");
  });
}

static int check_qk(const char* who, const ojx_qk_desc* d) {
  if (!d) return set_error(OJX_ERR_INVALID, "%s: desc is NULL", who);
  if (d->tokens < 0 || d->q_heads < 0 || d->kv_heads < 0)
    return set_error(OJX_ERR_INVALID, "%s: negative size", who);
  if (!known_dtype(d->dtype) || !known_dtype(d->dtype_weight))
    return set_error(OJX_ERR_INVALID, "%s: unknown dtype", who);
  if (d->head_dim < 2 || d->head_dim > 512 || d->head_dim % 2)
    return set_error(OJX_ERR_INVALID, "%s: head_dim %d is not an even number up to 512", who, d->head_dim);
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 2)
    return set_error(OJX_ERR_INVALID, "%s: rotary_dim %d is not an even number up to head_dim", who, d->rotary_dim);
  if (!(d->eps >= 0.0f)) return set_error(OJX_ERR_INVALID, "%s: eps must not be negative", who);
  if (d->table_rows < 0) return set_error(OJX_ERR_INVALID, "%s: negative size", who);
  if (d->tokens > 0 && ((d->q_heads && !d->q.data) || (d->kv_heads && !d->k.data) || !d->positions || (d->rotary_dim && !d->table)))
    return set_error(OJX_ERR_INVALID, "%s: NULL pointer", who);
  return OJX_OK;
}

static QkParams make_qk(const ojx_qk_desc* d) {
  QkParams p{};
  p.tokens = d->tokens;
  p.D = d->head_dim;
  p.rotary = d->rotary_dim;
  p.half = d->rotary_dim / 2;
  p.norm = 1;
  p.hq = d->q_heads;
  p.hk = d->kv_heads;
  p.dtype_w = d->dtype_weight;
  p.pos64 = d->positions_int64;
  p.eps = d->eps;
  p.inv_dim = 1.0f / d->head_dim;
  p.q = d->q.data, p.q_st = d->q.stride_t, p.q_sh = d->q.stride_h;
  p.k = d->k.data, p.k_st = d->k.stride_t, p.k_sh = d->k.stride_h;
  p.qw = d->q_weight;
  p.kw = d->k_weight;
  p.table = d->table;
  p.table_rows = d->table_rows;
  p.positions = d->positions;
  return p;
}

static bool qk_vector(const ojx_qk_desc* d) {
  const int es = dtype_size(d->dtype);
  return vector_pairs(d->head_dim, d->rotary_dim, d->interleaved != 0) && vector_rows(d->q, es) &&
         vector_rows(d->k, es) && aligned16(d->q_weight) && aligned16(d->k_weight);
}

// CTAs of a call (an equal share of its key tiles each, an SM each) and their workspace.
static int plan_tree(TaParams& p, int tile_rows, int unit, int D, cudaStream_t s, int* ctas) {
  const int rows = p.tokens * p.group;
  p.row_tiles = (rows + tile_rows - 1) / tile_rows;
  const int64_t per_seq = static_cast<int64_t>(p.cache.kv_heads) * p.row_tiles;
  const int64_t most = p.batch * per_seq * ((static_cast<int64_t>(p.width) * p.cache.page_size + unit - 1) / unit);
  if (per_seq > INT32_MAX || most > INT32_MAX) return set_error(OJX_ERR_INVALID, "ojx_tree_attention: too large");
  *ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, current_props().sm_count)));
  const size_t slots = static_cast<size_t>(*ctas) * 2 * tile_rows;
  char* ws = static_cast<char*>(stream_workspace(s, slots * (D * 4 + 8), 8, false));
  if (!ws) return workspace_error();
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + slots * D * 4);
  return OJX_OK;
}
template <int D>
static int join_tree(const TaParams& p, int tile_rows, int unit, int ctas, cudaStream_t s) {
  const int64_t all = static_cast<int64_t>(p.batch) * p.cache.kv_heads * p.tokens * p.group;
  // (launched while the attention kernel ends: what it reads of the call's inputs overlaps.
  // Not so in a capture: ojx_graph_capture_end orders the recorded nodes by plain edges.)
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (s) cudaStreamIsCapturing(s, &capture);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((all + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = capture == cudaStreamCaptureStatusNone ? 1 : 0;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const int st = cuda_status(cudaLaunchKernelEx(&cfg, tree_attention_parts_kernel<D>, p, tile_rows, unit, ctas), "tree_attention parts launch");
  return st ? st : launched("tree_attention parts launch");
}

template <int FMT, int D, bool FEW>
static int launch_tree(TaParams& p, cudaStream_t s) {
  using L = TaLayout<FMT, D, FEW>;
  std::lock_guard<std::mutex> pair(pair_mutex());
  int ctas = 0, st = plan_tree(p, 16, L::UNIT, D, s, &ctas);
  if (st) return st;
  auto kern = tree_attention_kernel<FMT, D, FEW>;
  if ((st = ensure_smem_attr(reinterpret_cast<const void*>(kern), L::SMEM))) return st;
  kern<<<ctas, L::NW * 32, L::SMEM, s>>>(p, g_wait_budget.load());
  st = launched("tree_attention launch");
  return st ? st : join_tree<D>(p, 16, L::UNIT, ctas, s);
}

template <int FMT, int D, int QT>
static int launch_tree_tc(TaParams& p, cudaStream_t s) {
  using L = TcLayout<FMT, D, QT>;
  auto kern = tree_attention_tc_kernel<FMT, D, QT>;
  int st = ensure_smem_attr(reinterpret_cast<const void*>(kern), L::SMEM);
  if (st) return st;
  std::lock_guard<std::mutex> pair(pair_mutex());
  int ctas = 0;
  if ((st = plan_tree(p, QT * TC_BN, TC_BN, D, s, &ctas))) return st;
  // A TMA box holds rows of one page, so the page size decides its rows; the swizzle's
  // pattern spans eight.
  CUtensorMap tk{}, tv{};
  p.box_rows = 0;
  if (!L::QUANT && p.cache.page_size % 8 == 0) {
    int r = 64;
    while (p.cache.page_size % r) r /= 2;
    const CUtensorMapDataType dt = FMT == TA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int64_t all = p.cache.num_pages * p.cache.kv_heads * p.cache.page_size;
    if ((st = make_tmap_2d_sw128(&tk, dt, 2, p.cache.k, D, all, D * 2, 64, r))) return st;
    if ((st = make_tmap_2d_sw128(&tv, dt, 2, p.cache.v, D, all, D * 2, 64, r))) return st;
    p.box_rows = r;
  }
  kern<<<ctas, L::THREADS, L::SMEM, s>>>(tk, tv, p, g_wait_budget.load());
  if ((st = launched("tree_attention_tc launch"))) return st;
  return join_tree<D>(p, QT * TC_BN, TC_BN, ctas, s);
}

template <int FMT>
static int launch_tree_fmt(TaParams& p, cudaStream_t s) {
  // Times for eight sequences of up to 16000 keys, 8 key heads of 128, in us:
  //   up to 16 rows the kernel of warp MMAs, which is done when HBM is (16 rows f16 74, e4m3 72);
  //   beyond them it would pass over the keys again, and tcgen05's takes over, whose time
  //   hardly depends on the rows (16 rows f16 75, e4m3 137; 64 rows 81, 141);
  //   up to 8 rows without the second half of a fragment (e4m3, 8 rows 60; 16 rows 72);
  //   beyond 128 rows two tiles share a pass (132 rows f16: two 110, one after the other 146),
  //   below it they would halve a tile (96 rows f16: one 84, two 104).
  const int rows = p.tokens * p.group;
  if (rows > 16) {
    const bool two = rows > 128;
    if (p.cache.head_dim == 64) return two ? launch_tree_tc<FMT, 64, 2>(p, s) : launch_tree_tc<FMT, 64, 1>(p, s);
    return two ? launch_tree_tc<FMT, 128, 2>(p, s) : launch_tree_tc<FMT, 128, 1>(p, s);
  }
  const bool few = rows <= 8;
  if (p.cache.head_dim == 64) return few ? launch_tree<FMT, 64, true>(p, s) : launch_tree<FMT, 64, false>(p, s);
  return few ? launch_tree<FMT, 128, true>(p, s) : launch_tree<FMT, 128, false>(p, s);
}

}  // namespace ojx

using namespace ojx;

extern "C" {

int ojx_qk_norm_rope(const ojx_qk_desc* d, void* q_out, void* k_out, ojx_stream s) {
  NvtxRange nvtx("ojx_qk_norm_rope");
  int st = check_qk("ojx_qk_norm_rope", d);
  if (st) return st;
  if (d->tokens == 0 || d->q_heads + d->kv_heads == 0) return OJX_OK;
  if ((d->q_heads && !q_out) || (d->kv_heads && !k_out))
    return set_error(OJX_ERR_INVALID, "ojx_qk_norm_rope: NULL output");
  QkParams p = make_qk(d);
  p.q_out = q_out;
  p.k_out = k_out;
  const bool vec = qk_vector(d) && aligned16(q_out) && aligned16(k_out);
  return launch_rows(p, d->dtype, vec, d->interleaved != 0, static_cast<cudaStream_t>(s));
}

int ojx_qkv_to_cache(const ojx_qk_desc* d, const ojx_rows* v, void* q_out, const ojx_kv_cache* cache,
                     const void* slots, int32_t slots_int64, ojx_stream s) {
  NvtxRange nvtx("ojx_qkv_to_cache");
  int st = check_qk("ojx_qkv_to_cache", d);
  if (st) return st;
  if ((st = check_cache("ojx_qkv_to_cache", cache))) return st;
  if (cache->head_dim != d->head_dim || cache->kv_heads != d->kv_heads)
    return set_error(OJX_ERR_INVALID, "ojx_qkv_to_cache: the cache holds %d heads of %d, the keys have %d of %d",
                     cache->kv_heads, cache->head_dim, d->kv_heads, d->head_dim);
  if (d->tokens == 0) return OJX_OK;
  if (!v || !v->data || !slots || (d->q_heads && !q_out))
    return set_error(OJX_ERR_INVALID, "ojx_qkv_to_cache: NULL pointer");
  QkParams p = make_qk(d);
  p.hv = d->kv_heads;
  p.v = v->data, p.v_st = v->stride_t, p.v_sh = v->stride_h;
  p.q_out = q_out;
  p.k_to_cache = 1;
  p.cache = *cache;
  p.slots = slots;
  p.slot64 = slots_int64;
  const bool vec = qk_vector(d) && vector_rows(*v, dtype_size(d->dtype)) && aligned16(q_out);
  return launch_rows(p, d->dtype, vec, d->interleaved != 0, static_cast<cudaStream_t>(s));
}

int ojx_qk_norm_rope_backward(const ojx_qk_desc* d, const ojx_rows* gq, const ojx_rows* gk, void* dq,
                              void* dk, void* dqw, void* dkw, ojx_stream stream) {
  NvtxRange nvtx("ojx_qk_norm_rope_backward");
  int st = check_qk("ojx_qk_norm_rope_backward", d);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t wbytes = static_cast<size_t>(d->head_dim) * dtype_size(d->dtype_weight);
  if (d->tokens == 0 || d->q_heads + d->kv_heads == 0) {  // no rows: the weights' sums are empty
    if (dqw && (st = cuda_status(cudaMemsetAsync(dqw, 0, wbytes, s), "clear dqw"))) return st;
    if (dkw && (st = cuda_status(cudaMemsetAsync(dkw, 0, wbytes, s), "clear dkw"))) return st;
    return OJX_OK;
  }
  if ((d->q_heads && (!gq || !gq->data || !dq)) || (d->kv_heads && (!gk || !gk->data || !dk)))
    return set_error(OJX_ERR_INVALID, "ojx_qk_norm_rope_backward: NULL pointer");
  QkParams p = make_qk(d);
  const int es = dtype_size(d->dtype);
  bool vec = qk_vector(d) && aligned16(dq) && aligned16(dk);
  if (gq) p.gq_data = gq->data, p.gq_st = gq->stride_t, p.gq_sh = gq->stride_h, vec = vec && vector_rows(*gq, es);
  if (gk) p.gk_data = gk->data, p.gk_st = gk->stride_t, p.gk_sh = gk->stride_h, vec = vec && vector_rows(*gk, es);
  p.dq = dq;
  p.dk = dk;
  const bool inter = d->interleaved != 0;
  p.npairs = p.D / (vec ? 16 : 2);
  p.lanes = std::min(32, pow2_at_least(p.npairs));
  p.gq = (p.hq + 32 / p.lanes - 1) / (32 / p.lanes);
  p.gk = (p.hk + 32 / p.lanes - 1) / (32 / p.lanes);
  // Blocks in proportion to each side's heads, at most one warp per token of it.
  const int64_t most = 2ll * current_props().sm_count;  // two blocks an SM
  auto blocks_of = [&](int heads) -> int64_t {
    if (heads == 0) return 0;
    const int64_t share = std::max<int64_t>(1, most * heads / (d->q_heads + d->kv_heads));
    return std::min(share, (d->tokens + 7) / 8);
  };
  p.q_blocks = static_cast<int>(blocks_of(d->q_heads));
  const int blocks = p.q_blocks + static_cast<int>(blocks_of(d->kv_heads));
  std::lock_guard<std::mutex> pair(pair_mutex());
  p.partial = static_cast<float*>(stream_workspace(s, static_cast<size_t>(blocks) * p.D * 4, 9, false));
  if (!p.partial) return workspace_error();
  int smem = 8 * p.D * 4;
  const int sms = current_props().sm_count, per_warp = 32 / p.lanes;
  // (streamed / prefetched as above: 800 tokens 10.2 / 9.5 us, 1200 11.9 / 12.0, 2400 16.7 / 19.1)
  const bool stream_rows = vec && p.tokens >= 8ll * sms && aligned16(p.table) && p.rotary % 4 == 0 &&
                           side_by_side(p.q_sh, p.D, p.hq) && side_by_side(p.k_sh, p.D, p.hk) && side_by_side(p.gq_sh, p.D, p.hq) &&
                           side_by_side(p.gk_sh, p.D, p.hk);
  const int heads_each = per_warp * (es == 4 ? 1 : 2);
  const int slot = 2 * heads_each * p.D * es + p.rotary * 4;
  if (stream_rows) {
    p.gq = (p.hq + heads_each - 1) / heads_each;
    p.gk = (p.hk + heads_each - 1) / heads_each;
    if (p.tokens * std::max(p.gq, p.gk) > INT32_MAX) return set_error(OJX_ERR_INVALID, "too many rows for one call");
    smem = std::max(smem, 8 * QK_GRAD_RING * slot);
  }
  st = for_dtype(d->dtype, [&](auto t) {
    using T = decltype(t);
    if (stream_rows) {
      auto go = [&](auto kern) {
        int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
        if (r) return r;
        kern<<<blocks, 256, smem, s>>>(p, slot, g_wait_budget.load());
        return launched("qk_grad_stream launch");
      };
      return inter ? go(qk_grad_stream_kernel<T, true>) : go(qk_grad_stream_kernel<T, false>);
    }
    if (vec && !inter) qk_grad_fast_kernel<T, false><<<blocks, 256, smem, s>>>(p);
    else if (vec) qk_grad_fast_kernel<T, true><<<blocks, 256, smem, s>>>(p);
    else if (p.npairs <= 64 && !inter) qk_grad_kernel<T, 2, false><<<blocks, 256, smem, s>>>(p);
    else if (p.npairs <= 64) qk_grad_kernel<T, 2, true><<<blocks, 256, smem, s>>>(p);
    else if (!inter) qk_grad_kernel<T, 8, false><<<blocks, 256, smem, s>>>(p);
    else qk_grad_kernel<T, 8, true><<<blocks, 256, smem, s>>>(p);
    return launched("qk_grad launch");
  });
  if (st || (!dqw && !dkw)) return st;
  qk_grad_weight_kernel<<<dim3((p.D + 31) / 32, 2), dim3(32, 32), 0, s>>>(p.partial, p.q_blocks, blocks, p.D, dqw,
                                                                        dkw, d->dtype_weight);
  return launched("qk_grad_weight launch");
}

int ojx_kv_append(const ojx_kv_cache* cache, const ojx_rows* k, const ojx_rows* v, int32_t dtype,
                  int64_t n, const void* slots, int32_t slots_int64, ojx_stream s) {
  NvtxRange nvtx("ojx_kv_append");
  int st = check_cache("ojx_kv_append", cache);
  if (st) return st;
  if (n < 0) return set_error(OJX_ERR_INVALID, "ojx_kv_append: negative size");
  if (!known_dtype(dtype)) return set_error(OJX_ERR_INVALID, "ojx_kv_append: unknown dtype");
  if (n == 0) return OJX_OK;
  if (!k || !v || !k->data || !v->data || !slots) return set_error(OJX_ERR_INVALID, "ojx_kv_append: NULL pointer");
  QkParams p{};
  p.tokens = n;
  p.D = cache->head_dim;
  p.hk = p.hv = cache->kv_heads;
  p.k = k->data, p.k_st = k->stride_t, p.k_sh = k->stride_h;
  p.v = v->data, p.v_st = v->stride_t, p.v_sh = v->stride_h;
  p.k_to_cache = 1;
  p.cache = *cache;
  p.slots = slots;
  p.slot64 = slots_int64;
  const int es = dtype_size(dtype);
  return launch_rows(p, dtype, vector_rows(*k, es) && vector_rows(*v, es), false, static_cast<cudaStream_t>(s));
}

int ojx_kv_read(const ojx_kv_cache* cache, void* k_out, void* v_out, int32_t dtype, int64_t n,
                const void* slots, int32_t slots_int64, ojx_stream stream) {
  NvtxRange nvtx("ojx_kv_read");
  int st = check_cache("ojx_kv_read", cache);
  if (st) return st;
  if (n < 0) return set_error(OJX_ERR_INVALID, "ojx_kv_read: negative size");
  if (!known_dtype(dtype)) return set_error(OJX_ERR_INVALID, "ojx_kv_read: unknown dtype");
  if (n == 0) return OJX_OK;
  if (!k_out || !v_out || !slots) return set_error(OJX_ERR_INVALID, "ojx_kv_read: NULL pointer");
  if (!aligned16(k_out) || !aligned16(v_out))
    return set_error(OJX_ERR_INVALID, "ojx_kv_read: outputs must be 16-byte aligned");
  const int64_t per_block = 2 * (256 / (cache->head_dim / 8));
  const int64_t grid = (n * cache->kv_heads + per_block - 1) / per_block;
  if (grid > INT32_MAX) return set_error(OJX_ERR_INVALID, "ojx_kv_read: too many rows for one call");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    kv_read_kernel<T><<<static_cast<unsigned>(grid), 256, 0, s>>>(*cache, slots, slots_int64, n,
                                                                  static_cast<T*>(k_out), static_cast<T*>(v_out));
    return launched("kv_read launch");
  });
}

int ojx_kv_keep_path(const ojx_kv_cache* cache, const int32_t* page_table, int32_t table_width,
                     const int32_t* context_lens, const int32_t* path, const int32_t* count,
                     int64_t batch, int32_t tokens, ojx_stream s) {
  NvtxRange nvtx("ojx_kv_keep_path");
  int st = check_cache("ojx_kv_keep_path", cache);
  if (st) return st;
  if (batch < 0 || tokens < 0 || table_width < 0)
    return set_error(OJX_ERR_INVALID, "ojx_kv_keep_path: negative size");
  if (batch == 0 || tokens == 0) return OJX_OK;
  if (!page_table || !context_lens || !path || !count)
    return set_error(OJX_ERR_INVALID, "ojx_kv_keep_path: NULL pointer");
  if (batch * cache->kv_heads > INT32_MAX) return set_error(OJX_ERR_INVALID, "ojx_kv_keep_path: too many heads");
  kv_keep_path_kernel<<<static_cast<unsigned>(batch * cache->kv_heads), 128, 0, static_cast<cudaStream_t>(s)>>>(
      *cache, page_table, table_width, context_lens, path, count, tokens);
  return launched("kv_keep_path launch");
}

int ojx_tree_attention(const ojx_tree_attention_desc* d, ojx_stream stream) {
  NvtxRange nvtx("ojx_tree_attention");
  if (!d) return set_error(OJX_ERR_INVALID, "ojx_tree_attention: desc is NULL");
  int st = check_cache("ojx_tree_attention", &d->cache);
  if (st) return st;
  const ojx_kv_cache& c = d->cache;
  if (c.head_dim != 64 && c.head_dim != 128)
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: head_dim %d is not 64 or 128", c.head_dim);
  if (d->dtype != OJX_BF16 && d->dtype != OJX_F16)
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: queries are bf16 or fp16");
  if (c.format < OJX_KV_INT8 && c.format != d->dtype)
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: a 16-bit cache has the queries' dtype");
  if (d->batch < 0 || d->tokens < 0 || d->q_heads < 0 || d->table_width < 0)
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: negative size");
  if (d->q_heads % c.kv_heads)
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: %d query heads do not share %d key heads evenly",
                     d->q_heads, c.kv_heads);
  if (!(d->scale > 0.0f)) return set_error(OJX_ERR_INVALID, "ojx_tree_attention: scale must be positive");
  if (d->batch == 0 || d->tokens == 0 || d->q_heads == 0) return OJX_OK;
  if (!d->q || !d->out || !d->context_lens || (d->table_width > 0 && !d->page_table))
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: NULL pointer");
  if (!aligned16(d->out)) return set_error(OJX_ERR_INVALID, "ojx_tree_attention: out must be 16-byte aligned");
  if (static_cast<int64_t>(d->tokens) * d->q_heads > INT32_MAX / 2 ||
      static_cast<int64_t>(d->table_width) * c.page_size > INT32_MAX / 2 ||
      c.num_pages * c.page_size > INT32_MAX / c.kv_heads)
    return set_error(OJX_ERR_INVALID, "ojx_tree_attention: too large");
  TaParams p{};
  p.cache = c;
  p.q = d->q;
  p.out = d->out;
  p.q_sb = d->q_stride_b, p.q_st = d->q_stride_t, p.q_sh = d->q_stride_h;
  p.dtype = d->dtype, p.batch = d->batch, p.tokens = d->tokens, p.q_heads = d->q_heads;
  p.group = d->q_heads / c.kv_heads;
  p.page_table = d->page_table;
  p.width = d->table_width;
  p.contexts = d->context_lens;
  p.drafts = d->draft_lens;
  p.mask = d->mask;
  p.mask_sb = d->mask_stride_b;
  p.words = (d->tokens + 63) / 64;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (c.page_size == 1 << i) p.page_shift = i;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c.format == OJX_KV_F16) return launch_tree_fmt<TA_F16>(p, s);
  if (c.format == OJX_KV_BF16) return launch_tree_fmt<TA_BF16>(p, s);
  if (c.format == OJX_KV_INT8) return launch_tree_fmt<TA_INT8>(p, s);
  return launch_tree_fmt<TA_FP8>(p, s);
}

int ojx_verify_drafts(const ojx_verify_desc* d, ojx_stream stream) {
  NvtxRange nvtx("ojx_verify_drafts");
  if (!d) return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: desc is NULL");
  if (d->batch < 0 || d->tokens < 0 || d->vocab < 0)
    return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: negative size");
  if (!known_dtype(d->dtype)) return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: unknown dtype");
  if (d->batch == 0) return OJX_OK;
  if (d->tokens < 1 || d->tokens > VD_MAX_TOKENS)
    return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: 1 to %d nodes, not %d", VD_MAX_TOKENS, d->tokens);
  if (d->vocab < 1 || d->vocab > (1 << 20))  // (a bit per token, in one CTA's shared memory)
    return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: a vocabulary has 1 to %d tokens", 1 << 20);
  if (!d->target || !d->token_ids || !d->parents || !d->uniforms || !d->path || !d->count || !d->next_token)
    return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: NULL pointer");
  if (d->batch > INT32_MAX / VD_CLUSTER) return set_error(OJX_ERR_INVALID, "ojx_verify_drafts: too many sequences");
  VerifyParams p{};
  p.target = d->target, p.t_sb = d->target_stride_b, p.t_st = d->target_stride_t;
  p.draft = d->draft, p.d_sb = d->draft_stride_b, p.d_st = d->draft_stride_t;
  p.tokens = d->token_ids, p.parents = d->parents, p.uniforms = d->uniforms;
  p.path = d->path, p.count = d->count, p.next = d->next_token;
  p.T = d->tokens;
  p.V = d->vocab;
  // As many CTAs a sequence as run at once: two fit an SM, and what does not fit waits for
  // a whole cluster's walk (64 sequences of 131072 tokens: 33 us with eight, 26 with four).
  int cluster = VD_CLUSTER;
  while (cluster > 1 && static_cast<int64_t>(d->batch) * cluster > 2ll * current_props().sm_count) cluster /= 2;
  const int64_t share = vd_per_warp(p.V, cluster) * VD_WARPS;
  const int smem = d->draft ? 0 : static_cast<int>((share + 31) / 32 * 4);
  return for_dtype(d->dtype, [&](auto t) {
    auto kern = verify_drafts_kernel<decltype(t)>;
    int st = ensure_smem_attr(reinterpret_cast<const void*>(kern), 160 * 1024);
    if (st) return st;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(d->batch) * cluster);
    cfg.blockDim = dim3(VD_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    st = cuda_status(cudaLaunchKernelEx(&cfg, kern, p), "verify_drafts launch");
    return st ? st : launched("verify_drafts launch");
  });
}

}  // extern "C"
