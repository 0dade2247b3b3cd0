"""Serving operators: what a decoding step needs between its GEMMs.

    qk_norm_rope     RMS norm of each query and key head and the position rotation, one pass
                     (differentiable)
    qkv_to_cache     the same, with keys and values written to a paged cache
    KVCache          pages of keys and values in bf16, fp16, int8 or e4m3: append, read, keep_path
    tree_attention   attention of the newest tokens (one, a chunk, or a tree of drafts) over a cache
    verify_drafts    acceptance of drafted tokens against the target's probabilities

qk_norm_rope has a gradient (not for its table); the others have none, and refuse inputs that
require one with RuntimeError, except under torch.no_grad().
Every function takes device tensors of either kind, and returns the same kind: torchcl
handles (launched on torchcl's current stream) or torch CUDA tensors (launched on torch's
current stream of the current device; strided views are read in place when their last
dimension is dense).  Integer arguments beside handles may also be CPU tensors; they are
uploaded.  Calls are asynchronous.  An index that lies outside its range on the device is
skipped and reported as ValueError by the first torchcl.synchronize() or to_cpu() after the
call has run (both wait for torchcl's streams only: synchronise torch's before, for its calls).
The reference has no counterpart of these functions.
"""
from __future__ import annotations

import ctypes
import math
import threading

import torch

from torchcl import _lib as L
from torchcl.api import _get_buf, _get_dtype, _get_shape, _wrap_output, is_opencl_tensor, to_opencl
from torchcl.ops.engine import ojx_dtype
from torchcl.runtime import context as _ctx
from torchcl.runtime.context import get_queue
from torchcl.runtime.memory import CLBuffer, get_buffer_pool, note_use

_FORMAT_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "int8": torch.int8,
                  "float8": torch.float8_e4m3fn}
_INTS, _INT32, _INT64 = (torch.int32, torch.int64), (torch.int32,), (torch.int64,)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ref = ctypes.byref


# ── device arguments ──────────────────────────────────────────────────────────

def _cuda(t) -> bool:
    """Whether a call is one of torch CUDA tensors: those go through the compiled binding,
    which checks its arguments in the same order and with the same words.  The functions
    below serve handles."""
    return isinstance(t, torch.Tensor) and t.is_cuda


def _first(t) -> None:
    if not is_opencl_tensor(t):
        raise ValueError("expected a device tensor: a torchcl handle or a torch CUDA tensor")


def _strides(shape) -> tuple:
    out, acc = [], 1
    for d in reversed(shape):
        out.append(acc)
        acc *= max(int(d), 1)
    return tuple(reversed(out))


class _Arg:
    """Address, shape, strides and dtype of one handle, and what keeps it alive.  Index arrays
    may also be CPU tensors: they are uploaded."""

    __slots__ = ("ptr", "shape", "strides", "dtype", "keep")

    def __init__(self, t, name: str, dtypes=None):
        if dtypes in (_INTS, _INT32, _INT64) and isinstance(t, torch.Tensor) and not is_opencl_tensor(t) and not t.is_cuda:
            if t.dtype in dtypes:
                t = to_opencl(t)
        elif not is_opencl_tensor(t):
            raise ValueError(f"{name}: torch CUDA tensors and torchcl handles (or CPU tensors) cannot be mixed in one call")
        self.shape, self.dtype = _get_shape(t), _get_dtype(t)
        if dtypes is not None and self.dtype not in dtypes:
            raise ValueError(f"{name}: expected {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}")
        buf = _get_buf(t)
        self.ptr, self.strides, self.keep = buf.buffer, _strides(self.shape), (t, buf)


def _code(dtype, name: str) -> int:
    if dtype not in _FLOATS:
        raise ValueError(f"{name}: unsupported dtype; expected float32, bfloat16 or float16")
    return ojx_dtype(dtype)


def _no_gradient(what: str, *inputs) -> None:
    if torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in inputs):
        raise RuntimeError(f"{what} has no gradient: detach its inputs, or call it under torch.no_grad()")


def _empty(shape, dtype):
    """(handle, address) of a new dense output."""
    numel = math.prod(shape)
    buf = get_buffer_pool().allocate(numel * torch.empty(0, dtype=dtype).element_size(), dtype, tuple(shape))
    return _wrap_output(buf, tuple(shape), dtype), buf.buffer


def _rows(t, name):
    """_Arg, L.Rows and (tokens, heads, head_dim) of [..., heads, head_dim] rows, leading
    dimensions as one."""
    a = _Arg(t, name)
    if len(a.shape) < 3:
        raise ValueError(f"{name}: expected [tokens, heads, head_dim], got {a.shape}")
    return a, L.Rows(a.ptr, a.strides[-3], a.strides[-2]), (math.prod(a.shape[:-2]), *a.shape[-2:])


def _same_rows(sizes, name, want) -> None:
    if sizes != want:
        raise ValueError(f"{name}: shape does not match {list(want)} rows")


# ── norms and rotations ────────────────────────────────────────────────────────

def rope_table(positions: int, rotary_dim: int, theta: float = 10000.0) -> torch.Tensor:
    """float32 [positions, rotary_dim] on the CPU: the cosines, then the sines, of
    position * theta^(-2i / rotary_dim), computed in 64 bits and rounded once."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} is not an even number")
    freq = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1))
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _qk_desc(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    """(L.QkDesc, dtype of the rows, dtype of the weights, what must stay alive)."""
    _first(q)
    qa, qrows, (tokens, heads, dim) = _rows(q, "q")
    ka, krows, k_sizes = _rows(k, "k")
    _same_rows(k_sizes, "k", (tokens, k_sizes[1], dim))
    if ka.dtype != qa.dtype:
        raise ValueError("q and k must share a dtype")
    weights, weight_type = [None, None], None
    for i, (w, name) in enumerate(((q_weight, "q_weight"), (k_weight, "k_weight"))):
        if w is None:
            continue
        a = weights[i] = _Arg(w, name)
        if a.shape != (dim,):
            raise ValueError(f"{name}: shape {a.shape}, expected ({dim},)")
        if weight_type not in (None, a.dtype):
            raise ValueError("q_weight and k_weight must share a dtype")
        weight_type = a.dtype
    ta = _Arg(table, "table", (torch.float32,))
    if len(ta.shape) != 2 or ta.shape[1] > dim or ta.shape[1] % 2:
        raise ValueError(f"table: shape {ta.shape} is not [positions, rotary_dim] with an even rotary_dim <= {dim}")
    pa = _Arg(positions, "positions", _INTS)
    if math.prod(pa.shape) != tokens:
        raise ValueError(f"positions: {pa.shape} for {tokens} tokens")
    weight_type = weight_type or qa.dtype
    d = L.QkDesc()
    d.tokens, d.q_heads, d.kv_heads, d.head_dim, d.rotary_dim = tokens, heads, k_sizes[1], dim, ta.shape[1]
    d.interleaved, d.dtype, d.dtype_weight = int(bool(interleaved)), _code(qa.dtype, "q"), _code(weight_type, "q_weight")
    d.positions_int64, d.eps = int(pa.dtype == torch.int64), eps
    d.q, d.k = qrows, krows
    d.q_weight, d.k_weight = (w.ptr if w is not None else None for w in weights)
    d.table, d.table_rows, d.positions = ta.ptr, ta.shape[0], pa.ptr
    return d, qa.dtype, weight_type, (qa, ka, weights, ta, pa)


def _qk_forward(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    if _cuda(q):
        return L.torch_binding().qk_forward(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    d, dtype, _, keep = _qk_desc(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    q_out, qp = _empty(_get_shape(q), dtype)
    k_out, kp = _empty(_get_shape(k), dtype)
    L.check(L.lib().ojx_qk_norm_rope(_ref(d), qp, kp, get_queue()), "qk_norm_rope")
    return q_out, k_out


def _qk_backward(gq, gk, q, k, q_weight, k_weight, table, positions, eps, interleaved, want_weights=True):
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rope; the weights' None where not wanted."""
    if _cuda(q):
        return L.torch_binding().qk_backward(gq, gk, q, k, q_weight, k_weight, table, positions, eps, interleaved,
                                             want_weights)
    d, dtype, wdtype, keep = _qk_desc(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    ga, gq_rows, gq_sizes = _rows(gq, "grad of q")
    gb, gk_rows, gk_sizes = _rows(gk, "grad of k")
    _same_rows(gq_sizes, "grad of q", (d.tokens, d.q_heads, d.head_dim))
    _same_rows(gk_sizes, "grad of k", (d.tokens, d.kv_heads, d.head_dim))
    if ga.dtype != dtype or gb.dtype != dtype:
        raise ValueError("gradients must have the dtype of q and k")
    dq, dqp = _empty(_get_shape(q), dtype)
    dk, dkp = _empty(_get_shape(k), dtype)
    out, ptrs = [], []
    for w in (q_weight, k_weight):
        t, p = _empty((d.head_dim,), wdtype) if w is not None and want_weights else (None, None)
        out.append(t)
        ptrs.append(p)
    L.check(L.lib().ojx_qk_norm_rope_backward(_ref(d), _ref(gq_rows), _ref(gk_rows), dqp, dkp, *ptrs, get_queue()),
            "qk_norm_rope backward")
    return dq, dk, out[0], out[1]


def qk_norm_rope(q, k, q_weight, k_weight, table, positions, eps: float = 1e-6, interleaved: bool = False):
    """Norm and rotate query and key heads in one pass: for every row x of q and k,
    y = rotate(weight * x / sqrt(mean(x^2) + eps)).

    q [..., q_heads, head_dim] and k [..., kv_heads, head_dim] share their leading
    dimensions (the tokens) and a dtype (float32, bfloat16, float16); weights are
    [head_dim] or None (ones); table is rope_table(...) on the device, its width the
    number of rotated elements; positions holds one row of it per token (int32 or int64;
    a position outside the table gives NaN and ValueError at the next synchronize).
    Pairs are (i, i + rotary_dim/2), or (2i, 2i + 1) when `interleaved`.  Sums run in
    fp32; outputs are rounded once to the inputs' dtype.  Returns dense (q, k).
    Differentiable once in q, k and the weights (QKNormRopeFunction); a derivative of its
    gradient raises RuntimeError."""
    if _cuda(q):
        return L.torch_binding().qk_norm_rope(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    _no_gradient("qk_norm_rope's table", table)
    if torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in (q, k, q_weight, k_weight)):
        from torchcl.autograd import QKNormRopeFunction
        return QKNormRopeFunction.apply(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    return _qk_forward(q, k, q_weight, k_weight, table, positions, eps, interleaved)


def qkv_to_cache(q, k, v, q_weight, k_weight, table, positions, cache: "KVCache", slots, eps: float = 1e-6,
                 interleaved: bool = False):
    """qk_norm_rope for serving: returns the normed and rotated q; the normed and rotated
    k (unrounded) and v go straight into `cache` at `slots` ([tokens], int32 or int64;
    a negative slot skips the token's keys and values)."""
    if _cuda(q):
        return L.torch_binding().qkv_to_cache(q, k, v, q_weight, k_weight, table, positions, cache._address(q), slots, eps,
                                              interleaved)
    _no_gradient("qkv_to_cache", q, k, v, q_weight, k_weight, table)
    d, dtype, _, keep = _qk_desc(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    va, v_rows, v_sizes = _rows(v, "v")
    _same_rows(v_sizes, "v", (d.tokens, d.kv_heads, d.head_dim))
    if va.dtype != dtype:
        raise ValueError("q, k and v must share a dtype")
    sa = _Arg(slots, "slots", _INTS)
    if math.prod(sa.shape) != d.tokens:
        raise ValueError(f"slots: {sa.shape} for {d.tokens} tokens")
    q_out, qp = _empty(_get_shape(q), dtype)
    L.check(L.lib().ojx_qkv_to_cache(_ref(d), _ref(v_rows), qp, _ref(cache._use(_ctx.get_device(), False)), sa.ptr,
                                     int(sa.dtype == torch.int64), get_queue()), "qkv_to_cache")
    return q_out


# ── the cache ────────────────────────────────────────────────────────────────

_dropped: list = []  # (device, pages) of caches that are gone, which calls may still use
_dropped_lock = threading.RLock()  # reentrant: a finalizer runs wherever a collection starts


def _free_pages(pages) -> None:
    for buf in pages:
        if isinstance(buf, CLBuffer):
            get_buffer_pool().free(buf)


def _capturing() -> bool:
    return _ctx._capture_active or torch.cuda.is_current_stream_capturing()


def _give_back() -> None:
    """Return the pages of dropped caches to their allocators, once the device is done with
    them.  A capture allows no wait: then they stay until the next cache is made or dropped."""
    if not _dropped or _capturing():
        return
    with _dropped_lock:
        batch = list(_dropped)
        _dropped.clear()
    for device in {d for d, _ in batch}:
        torch.cuda.synchronize(device)
    for _, pages in batch:
        _free_pages(pages)


def _one_device(*tensors) -> None:
    where = {str(t.device) for t in tensors if t is not None}
    if len(where) > 1:
        raise ValueError(f"pages and steps on more than one device: {', '.join(sorted(where))}")


class KVCache:
    """Keys and values in pages [num_pages, kv_heads, page_size, head_dim].

    format "bfloat16" or "float16" stores rows as they are; "int8" and "float8" (e4m3)
    store eight bits an element and one float32 step per row (a head of a token):
    step = max|x| * (1/127 or 1/448, in float32), read back as stored * step.  A row with a NaN or an
    infinity reads back as NaN.  Token slot s is row s % page_size of page s // page_size;
    which pages make up a sequence is the caller's page table.  head_dim is a multiple of
    16 up to 512 (64 or 128 for tree_attention).

    The constructor takes zeroed pages from torchcl's pool (it returns when they are clear);
    from_pages wraps tensors that exist.  Dropping a cache whose pages were used on the other
    side's streams (torchcl's pages in calls on torch tensors, or torch's in calls on handles)
    waits for the device before the pages go back; during a graph capture they go back later.
    A graph of such calls needs the cache kept.  Calls that share a cache are ordered by their
    streams, as for any buffer; a slot given twice in one call holds one of the two."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, format: str = "int8"):
        if format not in _FORMAT_DTYPES:
            raise ValueError(f"unknown cache format {format!r}: one of {sorted(_FORMAT_DTYPES)}")
        if min(num_pages, page_size, kv_heads) < 1:
            raise ValueError("a cache has at least one page, row and head")
        if head_dim < 16 or head_dim > 512 or head_dim % 16:
            raise ValueError(f"head_dim {head_dim} is not a multiple of 16 up to 512")
        _give_back()
        pool = get_buffer_pool()
        rows = num_pages * page_size * kv_heads
        quantised = format in ("int8", "float8")
        data = rows * head_dim * (1 if quantised else 2)
        self._pages = []
        try:
            for nbytes in (data, data, *((rows * 4, rows * 4) if quantised else ())):
                self._pages.append(pool.allocate(nbytes))
                pool.zero_fill(self._pages[-1])
            if not _ctx._capture_active:  # calls on any stream may follow: the pages are clear by then
                L.check(L.lib().ojx_stream_synchronize(get_queue()), "KVCache")
        except Exception:
            _free_pages(self._pages)
            raise
        self._pages += [None] * (4 - len(self._pages))
        self._owned = True
        self._set(num_pages, page_size, kv_heads, head_dim, format)

    def __del__(self):
        try:
            if getattr(self, "_shared", False):
                with _dropped_lock:
                    _dropped.append((self._device, self._pages))
                _give_back()
            elif getattr(self, "_owned", False):
                _free_pages(self._pages)
        except Exception:
            pass

    @classmethod
    def from_pages(cls, k_pages, v_pages, k_scale=None, v_scale=None) -> "KVCache":
        """A cache over dense torch CUDA tensors: pages [num_pages, kv_heads, page_size,
        head_dim] of bfloat16, float16, int8 or float8_e4m3fn, and for the last two the
        steps, float32 [num_pages, kv_heads, page_size], none of them negative; all on one
        device."""
        formats = {v: k for k, v in _FORMAT_DTYPES.items()}
        for t, n in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.is_contiguous() and t.dim() == 4):
                raise ValueError(f"{n}: expected a dense 4-D CUDA tensor")
            if t.dtype not in formats:
                raise ValueError(f"{n}: dtype {t.dtype}, expected one of {[str(d) for d in formats]}")
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError("k_pages and v_pages must share shape and dtype")
        fmt = formats[k_pages.dtype]
        if (fmt in ("int8", "float8")) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("steps belong to 8-bit pages, and only to them")
        for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is not None and not (t.is_cuda and t.is_contiguous() and t.dtype == torch.float32
                                      and t.shape == k_pages.shape[:3]):
                raise ValueError(f"{n}: expected dense float32 {tuple(k_pages.shape[:3])}")
        _one_device(k_pages, v_pages, k_scale, v_scale)
        self = cls.__new__(cls)
        self._owned = False
        self._pages = [k_pages, v_pages, k_scale, v_scale]
        pages, heads, size, dim = k_pages.shape
        if min(pages, heads, size) < 1:
            raise ValueError("a cache has at least one page, row and head")
        if dim < 16 or dim > 512 or dim % 16:
            raise ValueError(f"head_dim {dim} is not a multiple of 16 up to 512")
        self._set(pages, size, heads, dim, fmt)
        return self

    def _set(self, num_pages, page_size, kv_heads, head_dim, format):
        self.num_pages, self.page_size, self.kv_heads = num_pages, page_size, kv_heads
        self.head_dim, self.format = head_dim, format
        self._device = _ctx.get_device() if self._owned else self._pages[0].device.index
        addr = [None if b is None else b.buffer if isinstance(b, CLBuffer) else b.data_ptr() for b in self._pages]
        self._pooled = any(isinstance(b, CLBuffer) for b in self._pages)
        self._desc = L.KVCacheDesc(*addr, num_pages, page_size, kv_heads, head_dim, L.KV_FORMATS[format])

        self._where = ctypes.addressof(self._desc)
        self._shared = False  # used by calls that its pages' allocator knows nothing of

    def _use(self, device: int, on_torch: bool) -> "L.KVCacheDesc":
        if device != self._device:
            raise ValueError(f"the cache is on cuda:{self._device}, the call on cuda:{device}")
        if self._pooled == on_torch:
            self._shared = True
        if self._pooled:
            for buf in self._pages:
                if buf is not None:
                    note_use(buf)  # a graph being captured must keep it
        return self._desc

    def _address(self, t) -> int:
        """For a call of the binding whose first tensor is t."""
        self._use(t.get_device(), True)
        return self._where

    def append(self, k, v, slots) -> None:
        """Write keys and values [tokens, kv_heads, head_dim] (float32, bfloat16 or
        float16) to `slots` ([tokens], int32 or int64; a negative slot is skipped)."""
        if _cuda(k):
            return L.torch_binding().kv_append(self._address(k), k, v, slots)
        _no_gradient("KVCache.append", k, v)
        _first(k)
        ka, k_rows, sizes = _rows(k, "k")
        va, v_rows, v_sizes = _rows(v, "v")
        if sizes[1:] != (self.kv_heads, self.head_dim):
            raise ValueError(f"k: rows {sizes[1:]}, the cache holds {(self.kv_heads, self.head_dim)}")
        _same_rows(v_sizes, "v", sizes)
        if va.dtype != ka.dtype:
            raise ValueError("k and v must share a dtype")
        n = sizes[0]
        sa = _Arg(slots, "slots", _INTS)
        if math.prod(sa.shape) != n:
            raise ValueError(f"slots: {sa.shape} for {n} tokens")
        L.check(L.lib().ojx_kv_append(_ref(self._use(_ctx.get_device(), False)), _ref(k_rows), _ref(v_rows), _code(ka.dtype, "k"), n,
                                      sa.ptr, int(sa.dtype == torch.int64), get_queue()), "KVCache.append")

    def read(self, slots, dtype: torch.dtype = torch.bfloat16):
        """(k, v), dense [tokens, kv_heads, head_dim] of `dtype`, as the cache holds them
        at `slots`; a negative slot gives zeros."""
        if _cuda(slots):
            return L.torch_binding().kv_read(self._address(slots), slots, dtype)
        _first(slots)
        code = _code(dtype, "dtype")
        sa = _Arg(slots, "slots", _INTS)
        n = math.prod(sa.shape)
        shape = (*sa.shape, self.kv_heads, self.head_dim)
        k, kp = _empty(shape, dtype)
        v, vp = _empty(shape, dtype)
        L.check(L.lib().ojx_kv_read(_ref(self._use(_ctx.get_device(), False)), kp, vp, code, n, sa.ptr, int(sa.dtype == torch.int64),
                                    get_queue()), "KVCache.read")
        return k, v

    def keep_path(self, page_table, context_lens, path, count) -> None:
        """After verify_drafts: move the accepted nodes' rows, at context_lens[b] +
        path[b][0..count[b]], to context_lens[b] + 0, 1, ...; the sequence then holds
        context_lens[b] + 1 + count[b] tokens."""
        if _cuda(path):
            return L.torch_binding().kv_keep_path(self._address(path), page_table, context_lens, path, count)
        _first(path)
        pa, ta = _Arg(path, "path", _INT32), _Arg(page_table, "page_table", _INT32)
        ca, na = _Arg(context_lens, "context_lens", _INT32), _Arg(count, "count", _INT32)
        if len(pa.shape) != 2 or len(ta.shape) != 2:
            raise ValueError("path is [batch, tokens] and page_table [batch, pages]")
        batch, tokens = pa.shape
        if ta.shape[0] != batch or ca.shape != (batch,) or na.shape != (batch,):
            raise ValueError(f"page_table {ta.shape}, context_lens {ca.shape}, count {na.shape} for {batch} sequences")
        L.check(L.lib().ojx_kv_keep_path(_ref(self._use(_ctx.get_device(), False)), ta.ptr, ta.shape[1], ca.ptr, pa.ptr, na.ptr, batch,
                                         tokens, get_queue()), "KVCache.keep_path")


# ── attention over the cache ─────────────────────────────────────────────────

def tree_mask(parents) -> torch.Tensor:
    """The ancestors of each node of draft trees, as tree_attention's mask: int64
    [..., tokens, ceil(tokens / 64)] on the CPU; bit j % 64 of word j / 64 of row i is set
    when node j is i or an ancestor of i.  parents [tokens] or [batch, tokens]; a negative
    parent starts a tree.  ValueError unless parents[i] < i."""
    p = torch.as_tensor(parents).cpu().long()
    tokens = p.shape[-1]
    rows = p.reshape(math.prod(p.shape[:-1]), tokens)
    if bool((rows >= torch.arange(tokens)).any()):
        raise ValueError("a node's parent must come before it")
    words = (tokens + 63) // 64
    out = torch.zeros(*rows.shape, words, dtype=torch.int64)
    at = torch.arange(rows.shape[0])
    for i in range(tokens):
        known = rows[:, i] >= 0
        out[known, i] = out[at[known], rows[known, i]]
        bit = 1 << (i % 64)
        out[:, i, i // 64] |= bit - (1 << 64) if i % 64 == 63 else bit
    return out.reshape(*p.shape, words)


def tree_attention(q, cache: KVCache, page_table, context_lens, mask=None, draft_lens=None,
                   scale: float | None = None):
    """softmax(scale q k^T) v of each sequence's newest tokens over its pages.

    q [batch, tokens, q_heads, head_dim], bfloat16 or float16 (a 16-bit cache has the same
    dtype); head h reads key head h // (q_heads / kv_heads).  Key position j of sequence b
    is row j % page_size of page page_table[b][j // page_size].  Query i sees positions
    0 .. context_lens[b] - 1 and, of the new tokens j < draft_lens[b] (default: all), which
    have been written at context_lens[b] + j, those whose bit is set in mask (tree_mask;
    [tokens, words] or [batch, tokens, words]) or, without a mask, j <= i.  tokens = 1
    without a mask is a decoding step.  Queries i >= draft_lens[b], and queries that see
    nothing, give zeros; nothing a query does not see reaches it, whatever it holds.
    Over float16 and 8-bit caches weights count with 11 bits, down to 2^-31 of a row's largest
    (times its value's step); bfloat16 caches keep 17.  Scratch comes from the library, so
    torchcl's capture_graph records the call and torch.cuda.graph does not (RuntimeError), as
    for qk_norm_rope's gradient.  Returns dense [batch, tokens, q_heads, head_dim]."""
    if _cuda(q):
        return L.torch_binding().tree_attention(q, cache._address(q), page_table, context_lens, mask, draft_lens, scale)
    _no_gradient("tree_attention", q)
    _first(q)
    qa = _Arg(q, "q", (torch.bfloat16, torch.float16))
    if len(qa.shape) != 4 or qa.shape[3] != cache.head_dim:
        raise ValueError(f"q: shape {qa.shape} is not [batch, tokens, q_heads, {cache.head_dim}]")
    batch, tokens, heads, dim = qa.shape
    if heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads do not share {cache.kv_heads} key heads evenly")
    ta, ca = _Arg(page_table, "page_table", _INT32), _Arg(context_lens, "context_lens", _INT32)
    if len(ta.shape) != 2 or ta.shape[0] != batch or ca.shape != (batch,):
        raise ValueError(f"page_table {ta.shape} and context_lens {ca.shape} for {batch} sequences")
    da = ma = None
    if draft_lens is not None:
        da = _Arg(draft_lens, "draft_lens", _INT32)
        if da.shape != (batch,):
            raise ValueError(f"draft_lens {da.shape} for {batch} sequences")
    if mask is not None:
        ma = _Arg(mask, "mask", _INT64)
        rows = (tokens, (tokens + 63) // 64)
        if ma.shape not in (rows, (batch, *rows)):
            raise ValueError(f"mask: shape {ma.shape} is neither {rows} nor {(batch, *rows)}")
    out, op = _empty(qa.shape, qa.dtype)
    d = L.TreeAttentionDesc()
    d.cache = cache._use(_ctx.get_device(), False)
    d.q, d.out = qa.ptr, op
    d.q_stride_b, d.q_stride_t, d.q_stride_h = qa.strides[:3]
    d.dtype, d.batch, d.tokens, d.q_heads = _code(qa.dtype, "q"), batch, tokens, heads
    d.page_table, d.table_width, d.context_lens = ta.ptr, ta.shape[1], ca.ptr
    d.draft_lens = da.ptr if da is not None else None
    if ma is not None:
        d.mask, d.mask_stride_b = ma.ptr, math.prod(ma.shape[1:]) if len(ma.shape) == 3 else 0
    d.scale = dim ** -0.5 if scale is None else scale
    L.check(L.lib().ojx_tree_attention(_ref(d), get_queue()), "tree_attention")
    return out


# ── verification ─────────────────────────────────────────────────────────────

def verify_drafts(target_probs, tokens, parents, uniforms, draft_probs=None):
    """Which drafts the target accepts, and the token that follows them.

    tokens and parents, int32 [batch, nodes]: node 0 is the root, node i > 0 carries
    tokens[b][i], drafted after node parents[b][i] < i (a negative token: no node).
    target_probs and draft_probs [batch, nodes, vocab] (float32, bfloat16 or float16)
    hold the target's and the draft's probabilities of the token after each node;
    without draft_probs a draft counts as certain (the draft's likeliest tokens).
    uniforms float32 [batch, nodes] in [0, 1): u_i decides node i, u_0 the next token.
    Nodes are tried in order, when their parent is the node reached; a rejection leaves
    max(p - q, 0) (or p without the token), renormalised, to the next child and finally to
    the next token.  Accepted tokens and the next one are distributed as the target's if the
    children of a node were drawn independently of one another from its row of draft_probs
    (twice the same token included; children drawn without replacement are not that), or,
    without draft_probs, were chosen without a look at uniforms.
    Returns int32 path [batch, nodes] (the root and the accepted nodes, then -1), count
    [batch] (accepted drafts) and next_token [batch] (-1: the row holds no probability).
    Sums are exact in units of 2^-38, so results do not depend on the launch shape."""
    if _cuda(target_probs):
        return L.torch_binding().verify_drafts(target_probs, tokens, parents, uniforms, draft_probs)
    _no_gradient("verify_drafts", target_probs, uniforms, draft_probs)
    _first(target_probs)
    pa = _Arg(target_probs, "target_probs")
    if len(pa.shape) != 3:
        raise ValueError(f"target_probs: shape {pa.shape} is not [batch, nodes, vocab]")
    batch, nodes, vocab = pa.shape
    qa = None
    if draft_probs is not None:
        qa = _Arg(draft_probs, "draft_probs")
        if qa.dtype != pa.dtype:
            raise ValueError("draft_probs: expected the dtype of target_probs")
        if qa.shape != pa.shape:
            raise ValueError(f"draft_probs: shape {qa.shape}, target_probs has {pa.shape}")
    xa, ra = _Arg(tokens, "tokens", _INT32), _Arg(parents, "parents", _INT32)
    ua = _Arg(uniforms, "uniforms", (torch.float32,))
    for a, n in ((xa, "tokens"), (ra, "parents"), (ua, "uniforms")):
        if a.shape != (batch, nodes):
            raise ValueError(f"{n}: shape {a.shape}, expected {(batch, nodes)}")
    path, path_p = _empty((batch, nodes), torch.int32)
    count, count_p = _empty((batch,), torch.int32)
    token, token_p = _empty((batch,), torch.int32)
    d = L.VerifyDesc()
    d.target, d.target_stride_b, d.target_stride_t = pa.ptr, pa.strides[0], pa.strides[1]
    if qa is not None:
        d.draft, d.draft_stride_b, d.draft_stride_t = qa.ptr, qa.strides[0], qa.strides[1]
    d.vocab, d.token_ids, d.parents, d.uniforms = vocab, xa.ptr, ra.ptr, ua.ptr
    d.path, d.count, d.next_token = path_p, count_p, token_p
    d.batch, d.tokens, d.dtype = batch, nodes, _code(pa.dtype, "target_probs")
    L.check(L.lib().ojx_verify_drafts(_ref(d), get_queue()), "verify_drafts")
    return path, count, token


__all__ = ["KVCache", "qk_norm_rope", "qkv_to_cache", "rope_table", "tree_attention", "tree_mask", "verify_drafts"]
