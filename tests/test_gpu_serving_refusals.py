"""What the serving operators refuse and how they fail: failures inside a gradient, derivatives
that do not exist, arguments, in the same words on torch tensors and on handles; and the gradient
on handles."""
import subprocess
import sys
import textwrap

import pytest
import torch

from conftest import PKG
from test_gpu_serving import pages_for, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from torchcl import serving
    return serving


def test_out_of_memory_inside_a_gradient():
    """The gradient runs on a thread of torch's that holds no Python lock: a failed workspace
    is an exception there, not the end of the process."""
    code = """
        import ctypes, sys
        sys.path.insert(0, {pkg!r})
        import torch
        from torchcl import _lib as L, serving
        m = L.torch_binding()
        names = ("ojx_qk_norm_rope", "ojx_qk_norm_rope_backward", "ojx_qkv_to_cache", "ojx_kv_append",
                 "ojx_kv_read", "ojx_kv_keep_path", "ojx_tree_attention", "ojx_verify_drafts", "ojx_last_error")
        entries = {{n: ctypes.cast(getattr(L.lib(), n), ctypes.c_void_p).value for n in names}}
        fails = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_void_p] * 8)(lambda *a: L.OJX_ERR_OOM)
        m.bind(dict(entries, ojx_qk_norm_rope_backward=ctypes.cast(fails, ctypes.c_void_p).value))
        q, k = (torch.ones(3, 2, 64, device="cuda", requires_grad=True) for _ in "qk")
        table, pos = serving.rope_table(8, 64).cuda(), torch.arange(3, device="cuda")
        out = serving.qk_norm_rope(q, k, None, None, table, pos)
        try:
            (out[0].sum() + out[1].sum()).backward()
        except (RuntimeError, MemoryError) as e:
            assert "qk_norm_rope backward" in str(e), e
        else:
            raise AssertionError("no error")
        one = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_void_p] * 4)(lambda *a: L.OJX_ERR_OOM)
        m.bind(dict(entries, ojx_qk_norm_rope=ctypes.cast(one, ctypes.c_void_p).value))
        try:
            serving.qk_norm_rope(q.detach(), k.detach(), None, None, table, pos)
        except MemoryError as e:
            assert "qk_norm_rope" in str(e), e
        else:
            raise AssertionError("no error")
        print("both raised")
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code.format(pkg=str(PKG)))], capture_output=True, text=True, timeout=250)
    assert r.returncode == 0 and "both raised" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-2000:])


def operands(S):
    q, k = rnd(1, 3, 4, 64, dtype=torch.bfloat16).cuda(), rnd(2, 3, 2, 64, dtype=torch.bfloat16).cuda()
    cache = S.KVCache.from_pages(*pages_for("int8", 4, 2, 16, 64))
    return q, k, S.rope_table(16, 64).cuda(), torch.arange(3, device="cuda"), cache


def test_derivatives_that_do_not_exist_are_refused(S):
    """tree_attention, the cache and verification have none; an input that wants one says so
    instead of losing it.  Without gradients recorded the same tensors are fine."""
    q, k, table, pos, cache = operands(S)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    pages, ctx = torch.arange(4).int().cuda()[None], torch.tensor([3], dtype=torch.int32, device="cuda")
    p, tok = torch.full((1, 2, 5), 0.2, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    u = torch.full((1, 2), 0.5, device="cuda")
    g = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    calls = [lambda: S.qkv_to_cache(g(q), k, k, w, w, table, pos, cache, pos), lambda: S.qkv_to_cache(q, g(k), k, w, w, table, pos, cache, pos),
             lambda: S.qkv_to_cache(q, k, g(k), w, w, table, pos, cache, pos), lambda: S.qkv_to_cache(q, k, k, g(w), w, table, pos, cache, pos),
             lambda: S.qkv_to_cache(q, k, k, w, g(w), table, pos, cache, pos), lambda: cache.append(g(k), k, pos),
             lambda: cache.append(k, g(k), pos), lambda: S.tree_attention(g(q)[None], cache, pages, ctx),
             lambda: S.verify_drafts(g(p), tok, tok, u), lambda: S.verify_drafts(p, tok, tok, u, draft_probs=g(p))]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(RuntimeError, match="no gradient"):
        S.qk_norm_rope(q, k, w, w, g(table), pos)


def test_forward_mode_is_refused(S):
    import torch.autograd.forward_ad as fwd
    q, k, table, pos, cache = operands(S)
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for call in (lambda: S.qk_norm_rope(dual, k, None, None, table, pos), lambda: S.qk_norm_rope(q, fwd.make_dual(k, k), None, None, table, pos),
                     lambda: S.tree_attention(dual[None], cache, torch.arange(4).int().cuda()[None], torch.tensor([3], dtype=torch.int32, device="cuda"))):
            with pytest.raises((RuntimeError, NotImplementedError), match="forward|no gradient|jvp"):
                call()


def test_gradients_on_handles(S):
    """The handles' form of the gradient: the bits of the torch form."""
    import torchcl
    from torchcl.serving import _qk_backward
    h = torchcl.to_opencl
    q, k, w = rnd(1, 9, 4, 64), rnd(2, 9, 2, 64), 1 + rnd(3, 64, scale=0.2)
    gq, gk, table, pos = rnd(4, 9, 4, 64), rnd(5, 9, 2, 64), S.rope_table(16, 64), torch.arange(9, dtype=torch.int32)
    got = _qk_backward(*map(h, (gq, gk, q, k, w, w, table)), pos, 1e-6, False)
    d = [t.cuda().requires_grad_() for t in (q, k, w, w.clone())]
    out = S.qk_norm_rope(*d, table.cuda(), pos.cuda())
    want = torch.autograd.grad(out, d, [gq.cuda(), gk.cuda()])
    assert all(torch.equal(torchcl.to_cpu(a), b.cpu()) for a, b in zip(got, want))


@pytest.mark.parametrize("used", ["both", "q", "k"])
def test_autograd_through_handles(S, used):
    """qk_norm_rope of handles that require a gradient, and of handles that do not."""
    import torchcl
    h = torchcl.to_opencl
    q, k, w = rnd(1, 9, 4, 64), rnd(2, 9, 2, 64), 1 + rnd(3, 64, scale=0.2)
    gq, gk, table, pos = rnd(4, 9, 4, 64), rnd(5, 9, 2, 64), S.rope_table(16, 64), torch.arange(9, dtype=torch.int32)
    pick = lambda pair: list(pair) if used == "both" else [pair[used == "k"]]  # noqa: E731
    d = [t.cuda().requires_grad_() for t in (q, k, w, w.clone())]
    want = torch.autograd.grad(pick(S.qk_norm_rope(*d, table.cuda(), pos.cuda())), d, [t.cuda() for t in pick((gq, gk))])
    ours = [h(t).requires_grad_() for t in (q, k, w, w.clone())]
    out = S.qk_norm_rope(*ours, h(table), h(pos))
    got = torch.autograd.grad(pick(out), ours, [h(t) for t in pick((gq, gk))])
    assert all(torch.equal(torchcl.to_cpu(a), b.cpu()) for a, b in zip(got, want))
    cache = S.KVCache(2, 16, 2, 64, "float16")
    for call in (lambda: cache.append(ours[1], ours[1], h(pos)), lambda: S.qk_norm_rope(h(q), h(k), None, None, h(table).requires_grad_(), h(pos))):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()


def _bad_calls(S, on, other, cache):
    """Calls that are refused, by what is wrong; `on` puts a CPU tensor where the call's tensors
    are, `other` where they are not."""
    f, i = (lambda *shape, dtype=torch.float16: on(torch.ones(*shape, dtype=dtype))), (lambda *shape, dtype=torch.int32: on(torch.zeros(*shape, dtype=dtype)))
    q, k, table, pos = f(3, 4, 64), f(3, 2, 64), f(8, 64, dtype=torch.float32), i(3)
    qk = lambda **kw: S.qk_norm_rope(**{**dict(q=q, k=k, q_weight=None, k_weight=None, table=table, positions=pos), **kw})  # noqa: E731
    qkv = lambda **kw: S.qkv_to_cache(**{**dict(q=q, k=k, v=k, q_weight=None, k_weight=None, table=table, positions=pos, cache=cache, slots=pos), **kw})  # noqa: E731
    tree = lambda **kw: S.tree_attention(**{**dict(q=f(2, 3, 4, 64), cache=cache, page_table=i(2, 4), context_lens=i(2)), **kw})  # noqa: E731
    keep = lambda **kw: cache.keep_path(**{**dict(page_table=i(2, 4), context_lens=i(2), path=i(2, 3), count=i(2)), **kw})  # noqa: E731
    p = f(2, 3, 9)
    verify = lambda **kw: S.verify_drafts(**{**dict(target_probs=p, tokens=i(2, 3), parents=i(2, 3), uniforms=f(2, 3, dtype=torch.float32)), **kw})  # noqa: E731
    f32 = torch.float32
    return {
        "q flat": lambda: qk(q=f(3, 64)), "q whole numbers": lambda: qk(q=i(3, 4, 64), k=i(3, 2, 64)), "k tokens": lambda: qk(k=f(4, 2, 64)),
        "k dim": lambda: qk(k=f(3, 2, 32)), "k dtype": lambda: qk(k=f(3, 2, 64, dtype=f32)), "weight shape": lambda: qk(q_weight=f(32)),
        "weights differ": lambda: qk(q_weight=f(64), k_weight=f(64, dtype=f32)), "weight whole": lambda: qk(q_weight=i(64)),
        "table dtype": lambda: qk(table=f(8, 64)), "table odd": lambda: qk(table=f(8, 63, dtype=f32)), "table wide": lambda: qk(table=f(8, 66, dtype=f32)),
        "table flat": lambda: qk(table=f(64, dtype=f32)), "positions count": lambda: qk(positions=i(4)), "positions dtype": lambda: qk(positions=f(3)),
        "eps": lambda: qk(eps=-1.0), "mixed": lambda: qk(k=other(torch.ones(3, 2, 64, dtype=torch.float16))), "dim": lambda: qk(q=f(3, 4, 514), k=f(3, 2, 514)),
        "v shape": lambda: qkv(v=f(3, 4, 64)), "v dtype": lambda: qkv(v=f(3, 2, 64, dtype=f32)), "slots count": lambda: qkv(slots=i(2)),
        "cache heads": lambda: qkv(k=f(3, 4, 64), v=f(3, 4, 64)), "append heads": lambda: cache.append(q, q, pos), "append v": lambda: cache.append(k, q, pos),
        "append v dtype": lambda: cache.append(k, f(3, 2, 64, dtype=f32), pos), "append slots": lambda: cache.append(k, k, i(5)),
        "append whole": lambda: cache.append(i(3, 2, 64), i(3, 2, 64), pos), "append slots dtype": lambda: cache.append(k, k, f(3)),
        "read dtype": lambda: cache.read(pos, dtype=torch.int32), "read slots": lambda: cache.read(f(3)),
        "path dtype": lambda: keep(path=i(2, 3, dtype=torch.int64)), "path flat": lambda: keep(path=i(2)), "path batch": lambda: keep(count=i(3)),
        "path pages": lambda: keep(page_table=i(3, 4)), "q single": lambda: tree(q=f(2, 3, 4, 64, dtype=f32)), "q dim": lambda: tree(q=f(2, 3, 4, 32)),
        "q heads": lambda: tree(q=f(2, 3, 5, 64)), "table batch": lambda: tree(page_table=i(3, 4)), "table long": lambda: tree(page_table=i(2, 4, dtype=torch.int64)),
        "contexts": lambda: tree(context_lens=i(3)), "drafts": lambda: tree(draft_lens=i(3)), "mask dtype": lambda: tree(mask=i(3, 1)),
        "mask shape": lambda: tree(mask=i(3, 2, dtype=torch.int64)), "mask batch": lambda: tree(mask=i(3, 3, 1, dtype=torch.int64)), "scale": lambda: tree(scale=0.0),
        "target flat": lambda: verify(target_probs=f(2, 9)), "target whole": lambda: verify(target_probs=i(2, 3, 9)), "draft dtype": lambda: verify(draft_probs=f(2, 3, 9, dtype=f32)),
        "draft shape": lambda: verify(draft_probs=f(2, 3, 8)), "tokens dtype": lambda: verify(tokens=i(2, 3, dtype=torch.int64)), "tokens shape": lambda: verify(tokens=i(2, 4)),
        "uniforms dtype": lambda: verify(uniforms=f(2, 3)), "uniforms shape": lambda: verify(uniforms=f(3, 2, dtype=f32)), "parents mixed": lambda: verify(uniforms=other(torch.ones(2, 3))),
    }


def test_both_kinds_of_tensors_are_refused_alike(S):
    import torchcl
    h, c = torchcl.to_opencl, lambda t: t.cuda()
    ours, theirs = S.KVCache(4, 16, 2, 64, "float16"), S.KVCache.from_pages(*pages_for("float16", 4, 2, 16, 64))
    handles, tensors = _bad_calls(S, h, c, ours), _bad_calls(S, c, h, theirs)
    differ = {}
    for what in handles:
        said = []
        for call in (handles[what], tensors[what]):
            with pytest.raises(ValueError) as e:
                call()
            said.append(str(e.value))
        if said[0] != said[1]:
            differ[what] = said
    assert not differ, differ
