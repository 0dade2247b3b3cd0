// torch_binding.cpp — the serving operators on torch CUDA tensors: argument checks, output
// allocation and the call of libojx's C entries on torch's current stream, without
// Python's share of the work (a small call spends ten times its kernel's duration there).
// torchcl/serving does the same in Python for torchcl handles; both refuse the same calls in
// the same words.
//
// The C entries are bound by address from the libojx that torchcl loaded, so this module
// links against torch only.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>
#include <new>
#include <sstream>
#include "../../include/ojx.h"

namespace {

struct Entries {
  decltype(&ojx_qk_norm_rope) qk_norm_rope = nullptr;
  decltype(&ojx_qk_norm_rope_backward) qk_norm_rope_backward = nullptr;
  decltype(&ojx_qkv_to_cache) qkv_to_cache = nullptr;
  decltype(&ojx_kv_append) kv_append = nullptr;
  decltype(&ojx_kv_read) kv_read = nullptr;
  decltype(&ojx_kv_keep_path) kv_keep_path = nullptr;
  decltype(&ojx_tree_attention) tree_attention = nullptr;
  decltype(&ojx_verify_drafts) verify_drafts = nullptr;
  decltype(&ojx_last_error) last_error = nullptr;
} g;

template <typename F>
void take(const py::dict& d, const char* name, F& f) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}

void bind_entries(const py::dict& d) {
  take(d, "ojx_qk_norm_rope", g.qk_norm_rope);
  take(d, "ojx_qk_norm_rope_backward", g.qk_norm_rope_backward);
  take(d, "ojx_qkv_to_cache", g.qkv_to_cache);
  take(d, "ojx_kv_append", g.kv_append);
  take(d, "ojx_kv_read", g.kv_read);
  take(d, "ojx_kv_keep_path", g.kv_keep_path);
  take(d, "ojx_tree_attention", g.tree_attention);
  take(d, "ojx_verify_drafts", g.verify_drafts);
  take(d, "ojx_last_error", g.last_error);
}

// (Both exceptions are plain C++: a gradient runs on an autograd thread that does not hold the
// interpreter's lock, and torch or pybind11 turns them into Python's where it does.)
[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

struct OutOfMemory : std::bad_alloc {  // MemoryError; RuntimeError from a gradient
  explicit OutOfMemory(std::string why) : why_(std::move(why)) {}
  const char* what() const noexcept override { return why_.c_str(); }
  std::string why_;
};

void check(int status, const char* what) {
  if (status == OJX_OK) return;
  const std::string msg = std::string(what) + ": " + g.last_error();
  if (status == OJX_ERR_INVALID) throw py::value_error(msg);
  if (status == OJX_ERR_OOM) throw OutOfMemory(msg);
  throw std::runtime_error(msg);
}

std::string shape_of(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}

int code_of(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kFloat: return OJX_F32;
    case at::kBFloat16: return OJX_BF16;
    case at::kHalf: return OJX_F16;
    default: refuse(std::string(name) + ": unsupported dtype; expected float32, bfloat16 or float16");
  }
}

void on_device(const at::Tensor& t, const char* name, const at::Device& device) {
  if (!t.is_cuda()) refuse(std::string(name) + ": torch CUDA tensors and torchcl handles (or CPU tensors) cannot be mixed in one call");
  if (t.device() != device) refuse(std::string(name) + ": tensor on another device than the first argument");
}

// The call's device: that of its first tensor, which must be the current one.
at::Device call_device(const at::Tensor& t) {
  if (!t.is_cuda()) refuse("expected a device tensor: a torchcl handle or a torch CUDA tensor");
  if (t.device().index() != c10::cuda::current_device())
    refuse("tensor on cuda:" + std::to_string(t.device().index()) + ", but the current device is cuda:" +
           std::to_string(c10::cuda::current_device()));
  return t.device();
}

at::Tensor dense_last(const at::Tensor& t) {
  return t.dim() && t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t;
}
// An index array: int32 or (where `wide`) int64, dense.
at::Tensor index_of(const at::Tensor& t, const char* name, const at::Device& device, bool wide) {
  on_device(t, name, device);
  if (t.scalar_type() != at::kInt && !(wide && t.scalar_type() == at::kLong))
    refuse(std::string(name) + ": expected " + (wide ? "int32 or int64" : "int32"));
  return t.contiguous();
}

// Rows [..., heads, dim] with the leading dimensions as one.
struct RowsOf {
  at::Tensor t;
  ojx_rows r;
  int64_t tokens, heads, dim;
};
RowsOf rows_of(const at::Tensor& x, const char* name, const at::Device& device) {
  on_device(x, name, device);
  if (x.dim() < 3) refuse(std::string(name) + ": expected [tokens, heads, head_dim], got " + shape_of(x.sizes()));
  RowsOf o;
  o.t = dense_last(x.dim() > 3 ? x.reshape({-1, x.size(-2), x.size(-1)}) : x);
  o.tokens = 1;
  for (int64_t i = 0; i + 2 < x.dim(); ++i) o.tokens *= x.size(i);
  o.heads = x.size(-2);
  o.dim = x.size(-1);
  o.r = ojx_rows{o.t.data_ptr(), o.t.stride(0), o.t.stride(1)};
  return o;
}
void same_rows(const RowsOf& o, const char* name, int64_t tokens, int64_t heads, int64_t dim) {
  if (o.tokens != tokens || o.heads != heads || o.dim != dim)
    refuse(std::string(name) + ": shape does not match [" + std::to_string(tokens) + ", " + std::to_string(heads) + ", " +
           std::to_string(dim) + "] rows");
}

using MaybeTensor = std::optional<at::Tensor>;

// Derivatives that `what` does not have: an input that wants one is refused, so that it is not
// left out without a word.
void no_tangent(const char* what, std::initializer_list<const at::Tensor*> inputs) {
  for (const at::Tensor* t : inputs)
    if (t && t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(std::string(what) + " has no forward-mode derivative");
}
void no_gradient(const char* what, std::initializer_list<const at::Tensor*> inputs) {
  no_tangent(what, inputs);
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : inputs)
    if (t && t->defined() && t->requires_grad())
      throw std::runtime_error(std::string(what) + " has no gradient: detach its inputs, or call it under torch.no_grad()");
}
const at::Tensor* some(const MaybeTensor& t) { return t ? &*t : nullptr; }

struct QkCall {
  ojx_qk_desc d{};
  RowsOf q, k;
  at::Tensor qw, kw, table, positions;
  at::ScalarType weight_type;
};
QkCall qk_call(const at::Tensor& q, const at::Tensor& k, const MaybeTensor& qw, const MaybeTensor& kw, const at::Tensor& table,
               const at::Tensor& positions, double eps, bool interleaved) {
  const at::Device dev = call_device(q);
  QkCall c;
  c.q = rows_of(q, "q", dev);
  c.k = rows_of(k, "k", dev);
  same_rows(c.k, "k", c.q.tokens, c.k.heads, c.q.dim);
  if (q.scalar_type() != k.scalar_type()) refuse("q and k must share a dtype");
  c.weight_type = q.scalar_type();
  bool given = false;
  for (int i = 0; i < 2; ++i) {
    const MaybeTensor& w = i ? kw : qw;
    const char* name = i ? "k_weight" : "q_weight";
    if (!w) continue;
    on_device(*w, name, dev);
    if (w->dim() != 1 || w->size(0) != c.q.dim)
      refuse(std::string(name) + ": shape " + shape_of(w->sizes()) + ", expected (" + std::to_string(c.q.dim) + ",)");
    if (given && w->scalar_type() != c.weight_type) refuse("q_weight and k_weight must share a dtype");
    c.weight_type = w->scalar_type();
    given = true;
    (i ? c.kw : c.qw) = w->contiguous();
  }
  on_device(table, "table", dev);
  if (table.scalar_type() != at::kFloat) refuse("table: expected float32");
  if (table.dim() != 2 || table.size(1) > c.q.dim || table.size(1) % 2)
    refuse("table: shape " + shape_of(table.sizes()) + " is not [positions, rotary_dim] with an even rotary_dim <= " + std::to_string(c.q.dim));
  c.table = table.contiguous();
  c.positions = index_of(positions, "positions", dev, true);
  if (c.positions.numel() != c.q.tokens)
    refuse("positions: " + shape_of(positions.sizes()) + " for " + std::to_string(c.q.tokens) + " tokens");
  c.d.tokens = c.q.tokens;
  c.d.q_heads = static_cast<int32_t>(c.q.heads);
  c.d.kv_heads = static_cast<int32_t>(c.k.heads);
  c.d.head_dim = static_cast<int32_t>(c.q.dim);
  c.d.rotary_dim = static_cast<int32_t>(table.size(1));
  c.d.interleaved = interleaved;
  c.d.dtype = code_of(q.scalar_type(), "q");
  c.d.dtype_weight = code_of(c.weight_type, "q_weight");
  c.d.positions_int64 = c.positions.scalar_type() == at::kLong;
  c.d.eps = static_cast<float>(eps);
  c.d.q = c.q.r;
  c.d.k = c.k.r;
  c.d.q_weight = c.qw.defined() ? c.qw.data_ptr() : nullptr;
  c.d.k_weight = c.kw.defined() ? c.kw.data_ptr() : nullptr;
  c.d.table = static_cast<const float*>(c.table.data_ptr());
  c.d.table_rows = c.table.size(0);
  c.d.positions = c.positions.data_ptr();
  return c;
}

ojx_stream stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
at::Tensor like(const at::Tensor& t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }
const ojx_kv_cache* cache_at(uintptr_t p) { return reinterpret_cast<const ojx_kv_cache*>(p); }

std::tuple<at::Tensor, at::Tensor> qk_forward(const at::Tensor& q, const at::Tensor& k, const MaybeTensor& qw, const MaybeTensor& kw,
                                              const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved) {
  const QkCall c = qk_call(q, k, qw, kw, table, positions, eps, interleaved);
  at::Tensor qo = like(q), ko = like(k);
  check(g.qk_norm_rope(&c.d, qo.data_ptr(), ko.data_ptr(), stream()), "qk_norm_rope");
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_backward(const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q,
                                                                       const at::Tensor& k, const MaybeTensor& qw, const MaybeTensor& kw,
                                                                       const at::Tensor& table, const at::Tensor& positions, double eps,
                                                                       bool interleaved, bool want_weights) {
  const QkCall c = qk_call(q, k, qw, kw, table, positions, eps, interleaved);
  const RowsOf a = rows_of(gq, "grad of q", q.device()), b = rows_of(gk, "grad of k", q.device());
  same_rows(a, "grad of q", c.q.tokens, c.q.heads, c.q.dim);
  same_rows(b, "grad of k", c.k.tokens, c.k.heads, c.k.dim);
  if (gq.scalar_type() != q.scalar_type() || gk.scalar_type() != q.scalar_type()) refuse("gradients must have the dtype of q and k");
  at::Tensor dq = like(q), dk = like(k), dqw, dkw;
  if (want_weights && c.qw.defined()) dqw = like(c.qw);
  if (want_weights && c.kw.defined()) dkw = like(c.kw);
  check(g.qk_norm_rope_backward(&c.d, &a.r, &b.r, dq.data_ptr(), dk.data_ptr(), dqw.defined() ? dqw.data_ptr() : nullptr,
                                dkw.defined() ? dkw.data_ptr() : nullptr, stream()),
        "qk_norm_rope backward");
  return {dq, dk, dqw, dkw};
}

// The gradient as a step of a graph (create_graph): its own derivative is refused, not
// silently left out.
struct QkGradOnce : torch::autograd::Function<QkGradOnce> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, const at::Tensor& gq, const at::Tensor& gk,
                                                const at::Tensor& q, const at::Tensor& k, const MaybeTensor& qw, const MaybeTensor& kw,
                                                const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved,
                                                bool weights) {
    auto [dq, dk, dqw, dkw] = qk_backward(gq, gk, q, k, qw, kw, table, positions, eps, interleaved, weights);
    auto kept = [&](const at::Tensor& t) { return t.defined() ? t : at::empty({0}, q.options()); };
    return {dq, dk, kept(dqw), kept(dkw)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    throw std::runtime_error("qk_norm_rope: differentiable once");
  }
};

struct QkFunction : torch::autograd::Function<QkFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                                                const MaybeTensor& qw, const MaybeTensor& kw, const at::Tensor& table,
                                                const at::Tensor& positions, double eps, bool interleaved) {
    ctx->save_for_backward({q, k, qw.value_or(at::Tensor()), kw.value_or(at::Tensor()), table, positions});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["weights"] = (qw && qw->requires_grad()) || (kw && kw->requires_grad());
    auto [qo, ko] = qk_forward(q, k, qw, kw, table, positions, eps, interleaved);
    return {qo, ko};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    auto maybe = [](const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    const at::Tensor gq = grads[0].defined() ? grads[0] : at::zeros_like(s[0], at::MemoryFormat::Contiguous);
    const at::Tensor gk = grads[1].defined() ? grads[1] : at::zeros_like(s[1], at::MemoryFormat::Contiguous);
    if (at::GradMode::is_enabled()) {
      auto out = QkGradOnce::apply(gq, gk, s[0], s[1], maybe(s[2]), maybe(s[3]), s[4], s[5], ctx->saved_data["eps"].toDouble(),
                                   ctx->saved_data["interleaved"].toBool(), ctx->saved_data["weights"].toBool());
      const bool w = ctx->saved_data["weights"].toBool();
      return {out[0], out[1], w && s[2].defined() ? out[2] : at::Tensor(), w && s[3].defined() ? out[3] : at::Tensor(),
              at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
    auto [dq, dk, dqw, dkw] = qk_backward(gq, gk, s[0], s[1], maybe(s[2]), maybe(s[3]), s[4], s[5], ctx->saved_data["eps"].toDouble(),
                                          ctx->saved_data["interleaved"].toBool(), ctx->saved_data["weights"].toBool());
    return {dq, dk, dqw, dkw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k, const MaybeTensor& qw, const MaybeTensor& kw,
                                                const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved) {
  no_tangent("qk_norm_rope", {&q, &k, some(qw), some(kw)});
  no_gradient("qk_norm_rope's table", {&table});
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || (qw && qw->requires_grad()) || (kw && kw->requires_grad()))) {
    auto out = QkFunction::apply(q, k, qw, kw, table, positions, eps, interleaved);
    return {out[0], out[1]};
  }
  return qk_forward(q, k, qw, kw, table, positions, eps, interleaved);
}

at::Tensor qkv_to_cache(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const MaybeTensor& qw, const MaybeTensor& kw,
                        const at::Tensor& table, const at::Tensor& positions, uintptr_t cache, const at::Tensor& slots, double eps,
                        bool interleaved) {
  no_gradient("qkv_to_cache", {&q, &k, &v, some(qw), some(kw), &table});
  const QkCall c = qk_call(q, k, qw, kw, table, positions, eps, interleaved);
  const RowsOf vr = rows_of(v, "v", q.device());
  same_rows(vr, "v", c.k.tokens, c.k.heads, c.k.dim);
  if (v.scalar_type() != q.scalar_type()) refuse("q, k and v must share a dtype");
  const at::Tensor s = index_of(slots, "slots", q.device(), true);
  if (s.numel() != c.q.tokens) refuse("slots: " + shape_of(slots.sizes()) + " for " + std::to_string(c.q.tokens) + " tokens");
  at::Tensor qo = like(q);
  check(g.qkv_to_cache(&c.d, &vr.r, qo.data_ptr(), cache_at(cache), s.data_ptr(), s.scalar_type() == at::kLong, stream()), "qkv_to_cache");
  return qo;
}

void kv_append(uintptr_t cache, const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots) {
  no_gradient("KVCache.append", {&k, &v});
  const ojx_kv_cache* c = cache_at(cache);
  const at::Device dev = call_device(k);
  const RowsOf kr = rows_of(k, "k", dev), vr = rows_of(v, "v", dev);
  if (kr.heads != c->kv_heads || kr.dim != c->head_dim)
    refuse("k: rows (" + std::to_string(kr.heads) + ", " + std::to_string(kr.dim) + "), the cache holds (" + std::to_string(c->kv_heads) +
           ", " + std::to_string(c->head_dim) + ")");
  same_rows(vr, "v", kr.tokens, kr.heads, kr.dim);
  if (v.scalar_type() != k.scalar_type()) refuse("k and v must share a dtype");
  const at::Tensor s = index_of(slots, "slots", dev, true);
  if (s.numel() != kr.tokens) refuse("slots: " + shape_of(slots.sizes()) + " for " + std::to_string(kr.tokens) + " tokens");
  check(g.kv_append(c, &kr.r, &vr.r, code_of(k.scalar_type(), "k"), kr.tokens, s.data_ptr(), s.scalar_type() == at::kLong, stream()),
        "KVCache.append");
}

std::tuple<at::Tensor, at::Tensor> kv_read(uintptr_t cache, const at::Tensor& slots, at::ScalarType dtype) {
  const ojx_kv_cache* c = cache_at(cache);
  const at::Device dev = call_device(slots);
  const int code = code_of(dtype, "dtype");
  const at::Tensor s = index_of(slots, "slots", dev, true);
  std::vector<int64_t> shape(slots.sizes().begin(), slots.sizes().end());
  shape.push_back(c->kv_heads);
  shape.push_back(c->head_dim);
  const auto opt = at::TensorOptions().dtype(dtype).device(dev);
  at::Tensor k = at::empty(shape, opt), v = at::empty(shape, opt);
  check(g.kv_read(c, k.data_ptr(), v.data_ptr(), code, s.numel(), s.data_ptr(), s.scalar_type() == at::kLong, stream()), "KVCache.read");
  return {k, v};
}

void kv_keep_path(uintptr_t cache, const at::Tensor& page_table, const at::Tensor& context_lens, const at::Tensor& path, const at::Tensor& count) {
  const at::Device dev = call_device(path);
  const at::Tensor p = index_of(path, "path", dev, false), t = index_of(page_table, "page_table", dev, false);
  const at::Tensor ctx = index_of(context_lens, "context_lens", dev, false), n = index_of(count, "count", dev, false);
  if (p.dim() != 2 || t.dim() != 2) refuse("path is [batch, tokens] and page_table [batch, pages]");
  const int64_t batch = p.size(0);
  if (t.size(0) != batch || ctx.dim() != 1 || ctx.size(0) != batch || n.dim() != 1 || n.size(0) != batch)
    refuse("page_table " + shape_of(t.sizes()) + ", context_lens " + shape_of(ctx.sizes()) + ", count " + shape_of(n.sizes()) + " for " +
           std::to_string(batch) + " sequences");
  const auto at = [](const at::Tensor& x) { return static_cast<const int32_t*>(x.data_ptr()); };
  check(g.kv_keep_path(cache_at(cache), at(t), static_cast<int32_t>(t.size(1)), at(ctx), at(p), at(n), batch, static_cast<int32_t>(p.size(1)),
                       stream()),
        "KVCache.keep_path");
}

at::Tensor tree_attention(const at::Tensor& q_in, uintptr_t cache, const at::Tensor& page_table, const at::Tensor& context_lens,
                          const MaybeTensor& mask, const MaybeTensor& draft_lens, std::optional<double> scale) {
  no_gradient("tree_attention", {&q_in});
  const ojx_kv_cache* c = cache_at(cache);
  const at::Device dev = call_device(q_in);
  if (q_in.scalar_type() != at::kBFloat16 && q_in.scalar_type() != at::kHalf) refuse("q: expected bfloat16 or float16");
  if (q_in.dim() != 4 || q_in.size(3) != c->head_dim)
    refuse("q: shape " + shape_of(q_in.sizes()) + " is not [batch, tokens, q_heads, " + std::to_string(c->head_dim) + "]");
  const at::Tensor q = dense_last(q_in);
  const int64_t batch = q.size(0), tokens = q.size(1), heads = q.size(2), words = (tokens + 63) / 64;
  if (heads % c->kv_heads)
    refuse(std::to_string(heads) + " query heads do not share " + std::to_string(c->kv_heads) + " key heads evenly");
  const at::Tensor t = index_of(page_table, "page_table", dev, false), ctx = index_of(context_lens, "context_lens", dev, false);
  if (t.dim() != 2 || t.size(0) != batch || ctx.dim() != 1 || ctx.size(0) != batch)
    refuse("page_table " + shape_of(page_table.sizes()) + " and context_lens " + shape_of(context_lens.sizes()) + " for " +
           std::to_string(batch) + " sequences");
  ojx_tree_attention_desc d{};
  at::Tensor dl, m;
  if (draft_lens) {
    dl = index_of(*draft_lens, "draft_lens", dev, false);
    if (dl.dim() != 1 || dl.size(0) != batch)
      refuse("draft_lens " + shape_of(draft_lens->sizes()) + " for " + std::to_string(batch) + " sequences");
    d.draft_lens = static_cast<const int32_t*>(dl.data_ptr());
  }
  if (mask) {
    on_device(*mask, "mask", dev);
    if (mask->scalar_type() != at::kLong) refuse("mask: expected int64");
    const bool each = mask->dim() == 3;
    if (!(each || mask->dim() == 2) || (each && mask->size(0) != batch) || mask->size(-2) != tokens || mask->size(-1) != words)
      refuse("mask: shape " + shape_of(mask->sizes()) + " is neither " + shape_of({tokens, words}) + " nor " + shape_of({batch, tokens, words}));
    m = mask->contiguous();
    d.mask = static_cast<const int64_t*>(m.data_ptr());
    d.mask_stride_b = each ? tokens * words : 0;
  }
  at::Tensor out = like(q_in);
  d.cache = *c;
  d.q = q.data_ptr();
  d.out = out.data_ptr();
  d.q_stride_b = q.stride(0), d.q_stride_t = q.stride(1), d.q_stride_h = q.stride(2);
  d.dtype = code_of(q.scalar_type(), "q");
  d.batch = static_cast<int32_t>(batch), d.tokens = static_cast<int32_t>(tokens), d.q_heads = static_cast<int32_t>(heads);
  d.page_table = static_cast<const int32_t*>(t.data_ptr());
  d.table_width = static_cast<int32_t>(t.size(1));
  d.context_lens = static_cast<const int32_t*>(ctx.data_ptr());
  d.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(c->head_dim)));
  check(g.tree_attention(&d, stream()), "tree_attention");
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_drafts(const at::Tensor& target, const at::Tensor& tokens, const at::Tensor& parents,
                                                             const at::Tensor& uniforms, const MaybeTensor& draft) {
  no_gradient("verify_drafts", {&target, &uniforms, some(draft)});
  const at::Device dev = call_device(target);
  if (target.dim() != 3) refuse("target_probs: shape " + shape_of(target.sizes()) + " is not [batch, nodes, vocab]");
  const at::Tensor p = dense_last(target);
  at::Tensor q;
  if (draft) {
    on_device(*draft, "draft_probs", dev);
    if (draft->scalar_type() != target.scalar_type()) refuse("draft_probs: expected the dtype of target_probs");
    if (draft->sizes() != target.sizes())
      refuse("draft_probs: shape " + shape_of(draft->sizes()) + ", target_probs has " + shape_of(target.sizes()));
    q = dense_last(*draft);
  }
  const int64_t batch = p.size(0), nodes = p.size(1);
  const at::Tensor x = index_of(tokens, "tokens", dev, false), r = index_of(parents, "parents", dev, false);
  on_device(uniforms, "uniforms", dev);
  if (uniforms.scalar_type() != at::kFloat) refuse("uniforms: expected float32");
  const at::Tensor u = uniforms.contiguous();
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>{x, "tokens"}, {r, "parents"}, {u, "uniforms"}})
    if (t.dim() != 2 || t.size(0) != batch || t.size(1) != nodes)
      refuse(std::string(name) + ": shape " + shape_of(t.sizes()) + ", expected " + shape_of({batch, nodes}));
  const auto opt = x.options();
  at::Tensor path = at::empty({batch, nodes}, opt), count = at::empty({batch}, opt), next = at::empty({batch}, opt);
  ojx_verify_desc d{};
  d.target = p.data_ptr();
  d.target_stride_b = p.stride(0), d.target_stride_t = p.stride(1);
  if (q.defined()) d.draft = q.data_ptr(), d.draft_stride_b = q.stride(0), d.draft_stride_t = q.stride(1);
  d.vocab = p.size(2);
  d.token_ids = static_cast<const int32_t*>(x.data_ptr());
  d.parents = static_cast<const int32_t*>(r.data_ptr());
  d.uniforms = static_cast<const float*>(u.data_ptr());
  d.path = static_cast<int32_t*>(path.data_ptr());
  d.count = static_cast<int32_t*>(count.data_ptr());
  d.next_token = static_cast<int32_t*>(next.data_ptr());
  d.batch = static_cast<int32_t>(batch), d.tokens = static_cast<int32_t>(nodes);
  d.dtype = code_of(p.scalar_type(), "target_probs");
  check(g.verify_drafts(&d, stream()), "verify_drafts");
  return {path, count, next};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind_entries);
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("qk_forward", &qk_forward);
  m.def("qk_backward", &qk_backward);
  m.def("qkv_to_cache", &qkv_to_cache);
  m.def("kv_append", &kv_append);
  m.def("kv_read", [](uintptr_t cache, const at::Tensor& slots, const py::object& dtype) {
    return kv_read(cache, slots, torch::python::detail::py_object_to_dtype(dtype));
  });
  m.def("kv_keep_path", &kv_keep_path);
  m.def("tree_attention", &tree_attention);
  m.def("verify_drafts", &verify_drafts);
}
