"""The serving operators on the GPU against plain 64-bit implementations: types, head
layouts, odd sizes, strides, lengths of zero and one, masks that leave a row empty,
non-finite values in hidden places, gradients against the formula and against differences.

Tolerances: `u` is one rounding to the output's type.  float32 sums of D terms, rsqrt and
a rotation stay below 32 float32 roundings of the pair's size (8 sequential and 6 tree
additions, rsqrt 2 ulp, three products, a difference)."""
import random

import numpy as np
import pytest
import torch

import serving_reference as ref
from serving_reference import ROUND

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def S():
    from torchcl import serving
    return serving


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def within(got, want, tol):
    got = got.cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp(min=1e-300)).max()):.3g} x tolerance"


# ── norms and rotations ────────────────────────────────────────────────────────

QK = [  # tokens, q heads, kv heads, dim, rotary, interleaved, dtype
    (1, 1, 1, 64, 64, False, "bf16"), (5, 32, 8, 128, 128, False, "bf16"), (3, 7, 1, 96, 48, False, "f32"),
    (17, 4, 4, 256, 256, False, "f16"), (2, 3, 1, 512, 128, False, "bf16"), (9, 5, 1, 96, 64, True, "bf16"),
    (300, 8, 2, 64, 32, True, "f32"), (4, 2, 2, 6, 4, False, "f32"), (5, 3, 1, 34, 20, True, "f16"),
    (5, 3, 1, 100, 36, False, "bf16"), (33, 2, 1, 128, 0, False, "f16"), (2, 1, 1, 2, 2, False, "f32"),
    (1537, 3, 2, 80, 40, False, "bf16"), (3, 1, 1, 510, 510, True, "f32"),
]


def qk_inputs(tokens, hq, hk, dim, rotary, dtype, seed=1):
    from torchcl.serving import rope_table
    dt = DT[dtype]
    table = rope_table(5000, rotary, 10000.0)
    pos = torch.randint(0, 5000, (tokens,), generator=torch.Generator().manual_seed(seed))
    return (rnd(seed, tokens, hq, dim, dtype=dt, scale=3.0), rnd(seed + 1, tokens, hk, dim, dtype=dt, scale=0.02),
            (1 + rnd(seed + 2, dim, scale=0.3)).to(dt), (1 + rnd(seed + 3, dim, scale=0.3)).to(dt), table, pos)


@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,inter,dtype", QK)
def test_qk_forward(S, tokens, hq, hk, dim, rotary, inter, dtype):
    q, k, qw, kw, table, pos = qk_inputs(tokens, hq, hk, dim, rotary, dtype)
    got = S.qk_norm_rope(*(t.cuda() for t in (q, k, qw, kw, table, pos)), interleaved=inter)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        want, size = ref.norm_rope(x, w, table, pos, interleaved=inter)
        assert y.dtype == x.dtype
        u = ROUND[y.dtype] if y.dtype != torch.float32 else 0.0
        within(y, want, u * want.abs() + 32 * F32 * size + (6e-8 if dtype == "f16" else 0.0))


@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,inter,dtype", QK)
def test_qk_backward(S, tokens, hq, hk, dim, rotary, inter, dtype):
    q, k, qw, kw, table, pos = qk_inputs(tokens, hq, hk, dim, rotary, dtype)
    gq, gk = rnd(8, *q.shape, dtype=q.dtype), rnd(9, *k.shape, dtype=q.dtype)
    d = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
    out = S.qk_norm_rope(*d, table.cuda(), pos.cuda(), interleaved=inter)
    got = torch.autograd.grad(out, d, [gq.cuda(), gk.cuda()])
    for x, w, g, dx, dw in ((q, qw, gq, got[0], got[2]), (k, kw, gk, got[1], got[3])):
        want, dwant, size, dsize = ref.norm_rope_grad(x, w, g, table, pos, interleaved=inter)
        u = ROUND[x.dtype] if x.dtype != torch.float32 else 0.0
        within(dx, want, u * want.abs() + 64 * F32 * size + (6e-8 if dtype == "f16" else 0.0))
        # a sum of n terms in float32: registers, warps, blocks; each run at most n long
        rows = x.shape[0] * x.shape[1]
        within(dw, dwant, u * dwant.abs() + (64 + rows) * F32 * dsize)


@pytest.mark.parametrize("weighted", [True, False])
def test_qk_gradient_in_a_graph(S, weighted):
    """create_graph changes no gradient, and a second derivative is refused."""
    q, k = rnd(1, 7, 4, 64).cuda().requires_grad_(), rnd(2, 7, 2, 64).cuda().requires_grad_()
    w = rnd(3, 64).cuda().requires_grad_() if weighted else None
    table, pos = S.rope_table(16, 64).cuda(), torch.arange(7, dtype=torch.int32).cuda()
    inputs = [t for t in (q, k, w) if t is not None]

    def loss():
        a, b = S.qk_norm_rope(q, k, w, None, table, pos)
        return (a * a * a).sum() + b.sum()

    plain = torch.autograd.grad(loss(), inputs)
    kept = torch.autograd.grad(loss(), inputs, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, kept))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(kept[0].sum(), q)


def test_qk_gradient_against_differences(S):
    """<grad, v> against (L(x + hv) - L(x - hv)) / 2h, L = sum(g y) of the float32 kernel.
    Error: h^2/6 L''' <= h^2 * |g| (third derivatives of a normalised row are O(1) for rows
    of unit size), plus 2 * 32 roundings of the outputs over 2h."""
    q, k, qw, kw, table, pos = qk_inputs(6, 3, 2, 64, 64, "f32")
    q, k = q / 3, k / 0.02
    gq, gk = rnd(8, *q.shape), rnd(9, *k.shape)
    x = [q, k, qw, kw]
    d = [t.cuda().requires_grad_(True) for t in x]
    out = S.qk_norm_rope(*d, table.cuda(), pos.cuda())
    grads = torch.autograd.grad(out, d, [gq.cuda(), gk.cuda()])
    h = 2.0 ** -7

    def loss(parts):
        a, b = S.qk_norm_rope(*(t.cuda() for t in parts), table.cuda(), pos.cuda())
        return float((a.cpu().double() * gq).sum() + (b.cpu().double() * gk).sum())

    for n in range(4):
        v = rnd(20 + n, *x[n].shape)
        v = v / v.norm()
        up, down = ([t + s * h * v if i == n else t for i, t in enumerate(x)] for s in (1, -1))
        diff = (loss(up) - loss(down)) / (2 * h)
        # the outputs' roundings are independent: their root of squares, not their sum
        noise = 32 * F32 * float(torch.cat([gq.flatten(), gk.flatten()]).norm()) * 4 / h
        assert abs(diff - float((grads[n].cpu().double() * v).sum())) <= h * h * float(gq.norm() + gk.norm()) + noise


def test_qk_strides_weights_positions(S):
    """Slices of a fused projection, expanded gradients, no weights, int32 positions,
    misaligned rows, more leading dimensions."""
    from torchcl.serving import rope_table
    x = rnd(3, 2, 6, 12, 128, dtype=torch.bfloat16)
    table, pos = rope_table(64, 128), torch.arange(12).reshape(2, 6).int()
    dev = x.cuda()
    q, k = S.qk_norm_rope(dev[:, :, :8], dev[:, :, 8:10], None, None, table.cuda(), pos.cuda())
    for part, y in ((x[:, :, :8], q), (x[:, :, 8:10], k)):
        want, size = ref.norm_rope(part.reshape(12, -1, 128), None, table, pos.reshape(-1))
        assert y.shape == part.shape and y.is_contiguous()
        within(y.reshape(want.shape), want, ROUND[torch.bfloat16] * want.abs() + 32 * F32 * size)
    odd = torch.empty(12 * 131 + 3, dtype=torch.bfloat16, device="cuda")[3:].as_strided((12, 1, 128), (131, 128, 1))
    odd.copy_(x.reshape(12, 12, 128)[:, :1])
    q, _ = S.qk_norm_rope(odd, odd, None, None, table.cuda(), pos.cuda())
    want, size = ref.norm_rope(x.reshape(12, 12, 128)[:, :1], None, table, pos.reshape(-1))
    within(q, want, ROUND[torch.bfloat16] * want.abs() + 32 * F32 * size)
    a = x.reshape(12, 12, 128)[:, :4].float().cuda().requires_grad_(True)
    b = x.reshape(12, 12, 128)[:, 4:5].float().cuda().requires_grad_(True)
    oq, ok = S.qk_norm_rope(a, b, None, None, table.cuda(), pos.cuda())
    da, db = torch.autograd.grad([oq.sum() + ok.sum()], [a, b])
    for part, d in ((a, da), (b, db)):
        p = part.detach().cpu()
        want, _, size, _ = ref.norm_rope_grad(p, None, torch.ones_like(p), table, pos.reshape(-1))
        within(d, want, 64 * F32 * size)


def test_qk_empty_zero_rows_and_bad_positions(S):
    import torchcl
    from torchcl.serving import rope_table
    table = rope_table(16, 64).cuda()
    w = torch.ones(64, device="cuda", requires_grad=True)
    e = torch.zeros(0, 2, 64, device="cuda", requires_grad=True)
    q, k = S.qk_norm_rope(e, e, w, w, table, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert q.shape == k.shape == (0, 2, 64)
    (dw,) = torch.autograd.grad(q.sum() + k.sum(), [w])
    assert (dw == 0).all()
    z = torch.zeros(3, 1, 64, device="cuda")
    q, _ = S.qk_norm_rope(z, z, w.detach(), None, table, torch.tensor([0, 1, 15], device="cuda"))
    assert (q == 0).all()
    one = torch.ones(3, 1, 64, device="cuda")
    q, _ = S.qk_norm_rope(one, one, None, None, table, torch.tensor([0, 16, -1], device="cuda"))
    assert torch.isfinite(q[0]).all() and torch.isnan(q[1:]).all()
    with pytest.raises(ValueError, match="out of range"):
        torch.cuda.synchronize()
        torchcl.synchronize()
    torchcl.synchronize()  # reported once


# ── the cache ────────────────────────────────────────────────────────────────

FORMATS = ["bfloat16", "float16", "int8", "float8"]


def pages_for(fmt, pages, heads, size, dim):
    dt = {"int8": torch.int8, "float8": torch.float8_e4m3fn}.get(fmt) or getattr(torch, fmt)
    es = 1 if fmt in ref.TOP else 2
    data = [torch.zeros(pages * heads * size * dim * es, dtype=torch.uint8, device="cuda").view(dt).reshape(pages, heads, size, dim)
            for _ in "kv"]
    return data + ([torch.zeros(pages, heads, size, device="cuda") for _ in "kv"] if es == 1 else [None, None])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,heads,dim,size", [(1, 1, 16, 1), (7, 3, 96, 5), (65, 8, 128, 16), (40, 2, 512, 64), (300, 4, 64, 32)])
def test_cache_append_read_is_exact(S, fmt, dtype, n, heads, dim, size):
    k, v = rnd(1, n, heads, dim, dtype=DT[dtype], scale=7.0), rnd(2, n, heads, dim, dtype=DT[dtype], scale=1e-3)
    pages = n // size + 2
    cache = S.KVCache.from_pages(*pages_for(fmt, pages, heads, size, dim))
    slots = torch.randperm(pages * size, generator=torch.Generator().manual_seed(3))[:n].cuda()
    cache.append(k.cuda(), v.cuda(), slots)
    for x, y in zip((k, v), cache.read(slots.int(), dtype=torch.float32)):
        assert torch.equal(y.cpu(), ref.stored(x, fmt)[0])
    for x, y in zip((k, v), cache.read(slots, dtype=torch.bfloat16)):
        assert torch.equal(y.cpu(), ref.stored(x, fmt)[0].bfloat16())


@pytest.mark.parametrize("fmt", ["int8", "float8"])
def test_cache_special_rows(S, fmt):
    """Zeros, tiny and huge rows, NaN and infinities, ties of the rounding, skipped slots."""
    x = torch.zeros(8, 1, 64)
    x[1] = 1e-45
    x[2] = torch.linspace(-3e38, 3e38, 64)
    x[3, 0, 5] = float("nan")
    x[4, 0, 6] = float("inf")
    x[5] = torch.arange(64).float() - 32
    x[5, 0, 0] = 127.0
    x[6] = (torch.arange(64).float() - 31.5) / 127
    x[6, 0, 0] = 1.0
    x[7] = 5.0
    cache = S.KVCache.from_pages(*pages_for(fmt, 2, 1, 8, 64))
    slots = torch.tensor([8, 1, 2, 3, 4, 5, 6, -1], device="cuda")
    cache.append(x.cuda(), -x.cuda(), slots)
    k, v = cache.read(slots, dtype=torch.float32)
    want = ref.stored(x, fmt)[0]
    want[7] = 0
    for got, w in ((k, want), (v, -want)):
        got = got.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(w))
        assert torch.equal(got.nan_to_num(nan=0.0), w.nan_to_num(nan=0.0))
    assert torch.isnan(k[3:5]).all()


def test_cache_strided_source_and_bad_slots(S):
    import torchcl
    x = rnd(4, 6, 5, 128, dtype=torch.bfloat16)
    cache = S.KVCache.from_pages(*pages_for("int8", 3, 2, 4, 128))
    slots = torch.tensor([0, 5, 2, 99, 11, 12], device="cuda")
    d = x.cuda()
    cache.append(d[:, :2], d[:, 3:], slots)
    with pytest.raises(ValueError, match="out of range"):
        torchcl.synchronize()
    k, v = cache.read(slots[:3], dtype=torch.float32)
    assert torch.equal(k.cpu(), ref.stored(x[:3, :2], "int8")[0])
    assert torch.equal(v.cpu(), ref.stored(x[:3, 3:], "int8")[0])
    k, _ = cache.read(slots[3:], dtype=torch.float32)
    assert torch.equal(k.cpu()[1], ref.stored(x[4, :2], "int8")[0])
    assert (k[0] == 0).all() and (k[2] == 0).all()
    with pytest.raises(ValueError):
        torchcl.synchronize()
    empty = torch.zeros(0, 2, 128, device="cuda")
    cache.append(empty, empty, slots[:0])
    assert cache.read(slots[:0])[0].shape == (0, 2, 128)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,hq,hk,dim,rotary,inter", [("bf16", 8, 2, 128, 128, False), ("f16", 3, 3, 64, 32, True), ("f32", 4, 1, 96, 96, False)])
def test_qkv_to_cache(S, fmt, dtype, hq, hk, dim, rotary, inter):
    """q as qk_norm_rope; k is the unrounded row quantised: at most one step from the
    64-bit row's (float8: one spacing, an eighth of the value), v exactly as append."""
    n, size = 37, 8
    from torchcl.serving import rope_table
    x = rnd(5, n, hq + 2 * hk, dim, dtype=DT[dtype], scale=2.0)
    qw, kw = (1 + rnd(6, dim, scale=0.2)).to(DT[dtype]), (1 + rnd(7, dim, scale=0.2)).to(DT[dtype])
    table, pos = rope_table(100, rotary), torch.arange(n) + 50
    cache = S.KVCache.from_pages(*pages_for(fmt, 6, hk, size, dim))
    slots = torch.randperm(48, generator=torch.Generator().manual_seed(1))[:n]
    slots[4] = -1
    d = x.cuda()
    args = (qw.cuda(), kw.cuda(), table.cuda(), pos.cuda())
    q = S.qkv_to_cache(d[:, :hq], d[:, hq:hq + hk], d[:, hq + hk:], *args, cache, slots.cuda(), interleaved=inter)
    same, _ = S.qk_norm_rope(d[:, :hq], d[:, hq:hq + hk], *args, interleaved=inter)
    assert torch.equal(q, same)
    k, v = cache.read(slots.cuda(), dtype=torch.float32)
    want_v = ref.stored(x[:, hq + hk:], fmt)[0]
    want_v[4] = 0
    assert torch.equal(v.cpu(), want_v)
    want, size_ = ref.norm_rope(x[:, hq:hq + hk], kw, table, pos, interleaved=inter)
    amax = want.abs().amax(-1, keepdim=True)
    step = {"int8": 0.5 * amax / 127, "float8": want.abs() / 16 + amax / 448 * 2.0 ** -10}.get(fmt)
    if step is None:
        step = ROUND[getattr(torch, fmt)] * want.abs()
    tol = step * 1.001 + 64 * F32 * (size_ + amax)
    want[4], tol[4] = 0, 1e-30
    within(k, want, tol)


@pytest.mark.parametrize("fmt", FORMATS)
def test_keep_path(S, fmt):
    b, t, heads, dim, size, width = 4, 9, 3, 64, 4, 8
    cache = S.KVCache.from_pages(*pages_for(fmt, b * width, heads, size, dim))
    table = torch.randperm(b * width, generator=torch.Generator().manual_seed(2)).reshape(b, width).int()
    ctx = torch.tensor([0, 3, 17, 5], dtype=torch.int32)
    at = ctx[:, None] + torch.arange(t)
    slots = torch.gather(table, 1, (at // size).long()) * size + at % size
    x = rnd(6, b * t, heads, dim)
    cache.append(x.cuda(), 2 * x.cuda(), slots.reshape(-1).cuda())
    paths = [[0], [0, 2, 3, 7], [0, 1, 2, 3], [0, 8]]
    path = torch.full((b, t), -1, dtype=torch.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = torch.tensor(p)
    count = torch.tensor([len(p) - 1 for p in paths], dtype=torch.int32)
    cache.keep_path(table.cuda(), ctx.cuda(), path.cuda(), count.cuda())
    k, v = cache.read(slots.reshape(-1).cuda(), dtype=torch.float32)
    want = ref.stored(x, fmt)[0].reshape(b, t, heads, dim)
    for i, p in enumerate(paths):
        for j, node in enumerate(p):
            assert torch.equal(k.cpu().reshape(want.shape)[i, j], want[i, node])
            assert torch.equal(v.cpu().reshape(want.shape)[i, j], 2 * want[i, node])


# ── attention ────────────────────────────────────────────────────────────────

def random_parents(rng, tokens):
    return [-1] + [rng.randrange(-1 if rng.random() < 0.1 else max(0, i - 6), i) for i in range(1, tokens)]


def attention_case(S, b, t, contexts, drafts, hq, hk, dim, dtype, fmt, size, mask="tree", seed=0, spoil=None, spare=0):
    """(out, 64-bit out, size of its terms) for random data; `spoil` puts non-finite values
    into every row that no query of any sequence sees, and into hidden drafts."""
    rng = random.Random(seed)
    keys = max(c + d for c, d in zip(contexts, drafts))
    width = max(1, (keys + size - 1) // size) + spare
    pages = pages_for(fmt, b * width + 1, hk, size, dim)
    cache = S.KVCache.from_pages(*pages)
    table = torch.randperm(b * width + 1, generator=torch.Generator().manual_seed(seed))[:b * width].reshape(b, width).int()
    every = torch.arange((b * width + 1) * size)
    x = rnd(seed + 1, len(every), hk, dim, dtype=DT[dtype]), rnd(seed + 2, len(every), hk, dim, dtype=DT[dtype])
    k, v = (ref.stored(a, fmt)[0] for a in x)
    q = rnd(seed + 3, b, t, hq, dim, dtype=DT[dtype], scale=2.0)
    if mask == "tree":
        words = S.tree_mask(torch.tensor([random_parents(rng, t) for _ in range(b)]))
    elif mask == "random":
        words = torch.randint(-2 ** 62, 2 ** 62, (b, t, (t + 63) // 64), generator=torch.Generator().manual_seed(seed))
        words[:, ::3] = 0  # rows that see no draft
    else:
        words = None
    scale = dim ** -0.5
    out, sizes, bad_slots = [], [], set(range(len(every)))
    for i in range(b):
        n = contexts[i] + drafts[i]
        at = torch.arange(n)
        slot = (table[i].long()[at // size] * size + at % size) if n else at
        vis = torch.zeros(t, n, dtype=torch.bool)
        vis[:drafts[i], :contexts[i]] = True
        tree = ref.words_to_bool(words[i], t) if words is not None else torch.ones(t, t).tril().bool()
        vis[:drafts[i], contexts[i]:] = tree[:drafts[i], :drafts[i]]
        bad_slots -= {int(slot[j]) for j in range(n) if vis[:, j].any()}
        if spoil is not None and drafts[i] > 1:  # one draft seen by some rows only
            j = contexts[i] + drafts[i] - 1
            for a, y in zip(x, (k, v)):
                a[slot[j], :, 3] = spoil
            k, v = (ref.stored(a, fmt)[0] for a in x)
        o, s = ref.attend(q[i], k[slot], v[slot], vis, scale)
        out.append(o)
        sizes.append(s)
    if spoil is not None:
        for s in bad_slots:
            for a in x:
                a[s] = spoil
    cache.append(x[0].cuda(), x[1].cuda(), every.cuda())
    got = S.tree_attention(q.cuda(), cache, table.cuda(), torch.tensor(contexts, dtype=torch.int32).cuda(),
                           mask=None if words is None else words.cuda(),
                           draft_lens=None if drafts == [t] * b else torch.tensor(drafts, dtype=torch.int32).cuda())
    return got, torch.stack(out), torch.stack(sizes)


def attention_tolerance(got, want, size):
    """One rounding of the output; weights of at least 11 bits (f16), and scores to
    float32 (exp of a score of size 40 turns its 2^-19 into that much): 2^-9 of the terms."""
    return ROUND[got.dtype] * want.abs() + 2.0 ** -9 * size + 1e-7


ATTEND = [  # contexts, drafts, tokens, q heads, kv heads, dim, dtype, page, mask
    ([0], [1], 1, 1, 1, 64, "bf16", 16, None), ([5], [1], 1, 4, 1, 128, "f16", 16, None),
    ([700, 0, 33], [1, 1, 1], 1, 8, 2, 128, "bf16", 16, None), ([64, 63, 65, 127], [1] * 4, 1, 5, 5, 64, "f16", 32, None),
    ([100, 7], [9, 9], 9, 4, 2, 128, "bf16", 8, "tree"), ([129, 1000], [13, 16], 16, 7, 1, 64, "f16", 7, "tree"),
    ([40, 3, 0], [48, 1, 47], 48, 8, 2, 128, "bf16", 64, "tree"), ([300], [64], 64, 8, 1, 128, "f16", 128, "tree"),
    ([200, 0], [70, 70], 70, 2, 1, 64, "bf16", 16, "random"), ([0, 0, 9], [5, 0, 3], 5, 2, 2, 128, "f16", 4, "random"),
    ([77], [130], 130, 3, 1, 128, "bf16", 16, None), ([2500], [2], 2, 16, 1, 64, "bf16", 256, "tree"),
    ([1300, 2, 128, 0, 640], [33, 7, 1, 40, 12], 40, 8, 2, 64, "f16", 16, "tree"), ([3000], [100], 100, 4, 2, 128, "bf16", 32, None),
    ([384, 900], [66, 65], 66, 2, 1, 128, "f16", 5, "random"), ([4100, 130], [16, 16], 16, 16, 2, 64, "bf16", 64, "tree"),
    ([126, 127, 128, 129], [2, 1, 5, 3], 5, 16, 1, 128, "bf16", 16, "tree"), ([0, 0], [0, 0], 9, 8, 1, 64, "f16", 3, None),
    ([1], [1], 1, 40, 1, 128, "bf16", 1, None), ([0, 0], [0, 0], 3, 2, 1, 64, "f16", 3, None),
]


@pytest.mark.parametrize("fmt", ["native", "int8", "float8"])
@pytest.mark.parametrize("contexts,drafts,t,hq,hk,dim,dtype,size,mask", ATTEND)
def test_attention(S, fmt, contexts, drafts, t, hq, hk, dim, dtype, size, mask):
    fmt = {"bf16": "bfloat16", "f16": "float16"}[dtype] if fmt == "native" else fmt
    got, want, size_ = attention_case(S, len(contexts), t, contexts, drafts, hq, hk, dim, dtype, fmt, size, mask)
    within(got, want, attention_tolerance(got, want, size_))
    assert (got.cpu()[size_ == 0] == 0).all()


@pytest.mark.parametrize("spoil", [float("nan"), float("inf")])
@pytest.mark.parametrize("fmt", ["bfloat16", "float16", "int8", "float8"])
@pytest.mark.parametrize("t,hq,hk", [(6, 4, 1), (20, 8, 1), (40, 8, 2)])
def test_attention_hidden_values_do_not_leak(S, fmt, spoil, t, hq, hk):
    """Rows beyond a sequence, unused pages, and a draft hidden from most rows hold NaN or
    infinities; rows that do not see them are finite and right."""
    dtype = "f16" if fmt == "float16" else "bf16"
    got, want, size = attention_case(S, 3, t, [20, 0, 70], [t, 3, t - 1], hq, hk, 64, dtype, fmt, 16, "tree", spoil=spoil, spare=1)
    fine = torch.isfinite(want)
    assert fine.any() and not fine.all()
    g = got.cpu().double()
    tol = attention_tolerance(got, want, size)
    assert ((g - want).abs()[fine] <= tol[fine]).all()
    # a visible spoiled value: the whole row where its key is not finite
    assert not torch.isfinite(g[~fine]).any()


@pytest.mark.parametrize("fmt", ["bfloat16", "int8", "float8"])
def test_attention_scales_of_any_size(S, fmt):
    """Steps from 1e-12 to 1e6 among one sequence's keys and values."""
    b, t, hq, hk, dim, n = 1, 3, 4, 1, 64, 200
    cache = S.KVCache.from_pages(*pages_for(fmt, 16, hk, 16, dim))
    k = rnd(1, n, hk, dim, dtype=torch.bfloat16)
    v = (rnd(2, n, hk, dim) * torch.logspace(-12, 6, n)[:, None, None]).bfloat16()
    k[150:] *= -20  # the large values get next to no weight from some rows
    q = rnd(3, b, t, hq, dim, dtype=torch.bfloat16, scale=2.0)
    cache.append(k.cuda(), v.cuda(), torch.arange(n).cuda())
    got = S.tree_attention(q.cuda(), cache, torch.arange(16).int()[None].cuda(), torch.tensor([n - t], dtype=torch.int32).cuda())
    vis = torch.ones(t, n).tril(n - t).bool()
    want, size = ref.attend(q[0], ref.stored(k, fmt)[0], ref.stored(v, fmt)[0], vis, dim ** -0.5)
    within(got[0], want, attention_tolerance(got, want, size))


@pytest.mark.parametrize("fmt", ["float16", "int8", "float8"])
@pytest.mark.parametrize("t,hq,hk,dim", [(6, 4, 1, 128), (12, 4, 1, 64), (24, 4, 1, 128), (40, 8, 2, 64), (40, 4, 1, 128)])
def test_attention_value_steps_far_apart(S, fmt, t, hq, hk, dim):
    """Every thirteenth value row is 2^20 times the others, and its key takes almost all of
    its weight away (a score about 40 below the others'): the output comes from the small
    rows, whose weights must keep their bits."""
    n = 300 + t
    cache = S.KVCache.from_pages(*pages_for(fmt, 32, hk, 16, dim))
    k, v = rnd(1, n, hk, dim, dtype=torch.float16), rnd(2, n, hk, dim, dtype=torch.float16, scale=2.0 ** -8)
    q = rnd(3, 1, t, hq, dim, dtype=torch.float16).abs()
    k[::13] = -50.0 / dim ** 0.5
    v[::13] *= 2.0 ** 20
    v[::13] = v[::13].clamp(-60000, 60000)
    cache.append(k.cuda(), v.cuda(), torch.arange(n).cuda())
    got = S.tree_attention(q.cuda(), cache, torch.arange(32).int()[None].cuda(), torch.tensor([n - t], dtype=torch.int32).cuda())
    vis = torch.ones(t, n).tril(n - t).bool()
    want, size = ref.attend(q[0], ref.stored(k, fmt)[0], ref.stored(v, fmt)[0], vis, dim ** -0.5)
    within(got[0], want, attention_tolerance(got, want, size))


def test_attention_strided_queries_and_shared_mask(S):
    cache = S.KVCache.from_pages(*pages_for("int8", 8, 2, 16, 128))
    x = rnd(1, 128, 2, 128, dtype=torch.bfloat16)
    cache.append(x.cuda(), x.cuda(), torch.arange(128).cuda())
    fused = rnd(2, 2, 5, 12, 128, dtype=torch.bfloat16).cuda()
    table = torch.arange(8).reshape(2, 4).int().cuda()
    ctx = torch.tensor([30, 59], dtype=torch.int32).cuda()
    words = S.tree_mask([-1, 0, 0, 1, 2]).cuda()
    a = S.tree_attention(fused[:, :, 2:10], cache, table, ctx, mask=words)
    b = S.tree_attention(fused[:, :, 2:10].contiguous(), cache, table, ctx, mask=words.expand(2, 5, 1).contiguous())
    assert torch.equal(a, b)


def test_attention_errors_on_the_device(S):
    import torchcl
    cache = S.KVCache.from_pages(*pages_for("int8", 2, 1, 16, 64))
    q = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for table, ctx in ((i32(7)[None], i32(3)), (i32(-1)[None], i32(3)), (i32(0)[None], i32(40))):
        S.tree_attention(q, cache, table, ctx)
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match="out of range"):
            torchcl.synchronize()


def test_attention_on_a_side_stream(S):
    """Work launched on torch's current stream: inputs made there, no host wait."""
    cache = S.KVCache.from_pages(*pages_for("int8", 8, 2, 16, 64))
    q = rnd(1, 2, 3, 4, 64, dtype=torch.bfloat16)
    x = rnd(2, 128, 2, 64, dtype=torch.bfloat16).cuda()
    table, ctx = torch.arange(8).reshape(2, 4).int().cuda(), torch.tensor([30, 50], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(x, x, torch.arange(128, device="cuda"))
        a = S.tree_attention(q.cuda(non_blocking=True), cache, table, ctx)
    side.synchronize()
    assert torch.equal(a, S.tree_attention(q.cuda(), cache, table, ctx))


# ── verification ─────────────────────────────────────────────────────────────

def verify_case(b, t, v, dtype, sampled, seed, chain=False, temperature=2.0):
    rng = random.Random(seed)
    parents = [[-1] + [i - 1 if chain else rng.randrange(max(0, i - 4), i) for i in range(1, t)] for _ in range(b)]
    logits = rnd(seed, b, t, v, scale=temperature)
    p = torch.softmax(logits, -1).to(DT[dtype])
    q = torch.softmax(logits + 0.8 * rnd(seed + 1, b, t, v), -1).to(DT[dtype])
    tokens = torch.zeros(b, t, dtype=torch.int32)
    for i in range(b):
        for j in range(1, t):
            row = q[i, parents[i][j]].float()
            tokens[i, j] = int(torch.multinomial(row, 1, generator=torch.Generator().manual_seed(seed + 31 * j + i))) if sampled \
                else int(row.topk(min(v, 3)).indices[rng.randrange(min(v, 3))])
    u = torch.rand(b, t, generator=torch.Generator().manual_seed(seed + 2))
    return p, tokens, torch.tensor(parents, dtype=torch.int32), u, q if sampled else None


def check_verify(S, p, tokens, parents, u, q):
    path, count, nxt = (x.cpu() for x in S.verify_drafts(p.cuda(), tokens.cuda(), parents.cuda(), u.cuda(),
                                                          draft_probs=None if q is None else q.cuda()))
    f = lambda x: x.float().numpy()  # noqa: E731
    for i in range(len(tokens)):
        want, token = ref.verify(f(p[i]), tokens[i].tolist(), parents[i].tolist(), u[i].numpy(), None if q is None else f(q[i]))
        assert path[i].tolist() == want + [-1] * (tokens.shape[1] - len(want))
        assert int(count[i]) == len(want) - 1 and int(nxt[i]) == token
    return count


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("b,t,v,dtype,chain", [
    (1, 1, 1, "f32", True), (3, 2, 7, "f32", True), (5, 6, 1000, "f32", True), (4, 24, 513, "f32", False),
    (9, 40, 131, "bf16", False), (3, 12, 4097, "f16", False), (2, 5, 40001, "f32", True), (40, 17, 64, "f32", False)])
def test_verify_against_reference(S, sampled, b, t, v, dtype, chain):
    counts = [check_verify(S, *verify_case(b, t, v, dtype, sampled, seed, chain)) for seed in (1, 2)]
    if sampled and t > 4 and b > 2:
        assert sum(int(c.sum()) for c in counts) > 0


def test_verify_edges(S):
    """Identical distributions always accept; disjoint ones never do, and draw from the
    target; padding, one-hot rows, non-finite and empty rows, bad indices, strided rows."""
    import torchcl
    p, tokens, parents, u, q = verify_case(6, 8, 300, "f32", True, 5, chain=True)
    assert check_verify(S, p, tokens, parents, u, p).tolist() == [7] * 6
    hot = torch.zeros_like(p)
    hot[..., 11] = 1.0
    tokens[:] = 11
    assert check_verify(S, hot, tokens, parents, u, None).tolist() == [7] * 6
    other = torch.zeros_like(p)
    other[..., 12] = 1.0
    assert check_verify(S, other, tokens, parents, u, hot).tolist() == [0] * 6
    tokens[:, 4:] = -1
    assert check_verify(S, hot, tokens, parents, u, None).tolist() == [3] * 6
    assert check_verify(S, torch.zeros_like(p), tokens, parents, u, None).tolist() == [0] * 6
    bad = p.clone()
    bad[:, :, ::7] = float("nan")
    bad[:, :, 1::7] = float("-inf")
    check_verify(S, bad, tokens, parents, u, None)
    wide = torch.zeros(6, 8, 320)
    wide[..., :300] = p
    a = S.verify_drafts(wide.cuda()[..., :300], tokens.cuda(), parents.cuda(), u.cuda())
    b = S.verify_drafts(p.cuda(), tokens.cuda(), parents.cuda(), u.cuda())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    torchcl.synchronize()
    tokens[0, 1], parents[1, 2] = 300, 5
    S.verify_drafts(p.cuda(), tokens.cuda(), parents.cuda(), u.cuda())
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="out of range"):
        torchcl.synchronize()


def test_verify_follows_the_target_distribution(S):
    """20,000 sequences with one row each way: the next emitted token (the first accepted
    draft, or the drawn one) has the target's frequencies.  5 sigma of a binomial share."""
    n, v = 20000, 8
    p = torch.softmax(rnd(1, v, scale=1.5), 0)
    q = torch.softmax(rnd(2, v, scale=1.5), 0)
    gen = torch.Generator().manual_seed(3)
    x = torch.multinomial(q, 2 * n, replacement=True, generator=gen).reshape(n, 2)
    tokens = torch.cat([torch.zeros(n, 1, dtype=torch.int64), x], 1).int()  # two siblings
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32).expand(n, 3).contiguous()
    rows = [a.expand(n, 3, v).contiguous().cuda() for a in (p, q)]
    path, count, nxt = S.verify_drafts(rows[0], tokens.cuda(), parents.cuda(), torch.rand(n, 3, generator=gen).cuda(), draft_probs=rows[1])
    first = torch.where(count.cpu() > 0, tokens.gather(1, path.cpu()[:, 1:2].clamp(min=0).long())[:, 0], nxt.cpu())
    share = torch.bincount(first.long(), minlength=v) / n
    assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()
    assert int(count.sum()) > n // 4


# ── handles ──────────────────────────────────────────────────────────────────

def test_handles_give_the_same_bits(S):
    """Every operator on torchcl handles, on torchcl's stream, as on torch tensors."""
    import torchcl
    q, k, qw, kw, table, pos = qk_inputs(6, 4, 2, 64, 64, "bf16")
    h = torchcl.to_opencl
    a = S.qk_norm_rope(*map(h, (q, k, qw, kw, table)), pos)
    b = S.qk_norm_rope(*(t.cuda() for t in (q, k, qw, kw, table, pos)))
    assert all(torch.equal(torchcl.to_cpu(x), y.cpu()) for x, y in zip(a, b))
    ours, theirs = S.KVCache(4, 8, 2, 64, "int8"), S.KVCache.from_pages(*pages_for("int8", 4, 2, 8, 64))
    slots = torch.tensor([3, 9, 30, 1, 0, 2], dtype=torch.int32)
    va = S.qkv_to_cache(*map(h, (q, k, k, qw, kw, table)), h(pos.int()), ours, h(slots))
    vb = S.qkv_to_cache(*(t.cuda() for t in (q, k, k, qw, kw, table, pos)), theirs, slots.cuda())
    assert torch.equal(torchcl.to_cpu(va), vb.cpu())
    ours.append(h(k), h(k), slots)
    theirs.append(k.cuda(), k.cuda(), slots.cuda())
    for x, y in zip(ours.read(h(slots)), theirs.read(slots.cuda())):
        assert torch.equal(torchcl.to_cpu(x), y.cpu())
    ptab, ctx, mask = torch.tensor([[0, 1], [3, 2]], dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32), S.tree_mask([-1, 0, 0])
    qq = rnd(4, 2, 3, 4, 64, dtype=torch.bfloat16)
    x = S.tree_attention(h(qq), ours, ptab, ctx, mask=mask)
    y = S.tree_attention(qq.cuda(), theirs, ptab.cuda(), ctx.cuda(), mask=mask.cuda())
    assert torch.equal(torchcl.to_cpu(x), y.cpu())
    p, tokens, parents, u, _ = verify_case(2, 3, 50, "f32", False, 3)
    got = S.verify_drafts(h(p), tokens, parents, h(u))
    want = S.verify_drafts(*(t.cuda() for t in (p, tokens, parents, u)))
    assert all(torch.equal(torchcl.to_cpu(a), b.cpu()) for a, b in zip(got, want))
    ours.keep_path(ptab, ctx, got[0], got[1])
    torchcl.synchronize()


def test_graph_capture_of_a_decoding_step(S):
    import torchcl
    from torchcl.jit.graph_runner import capture_graph
    cache = S.KVCache(8, 16, 2, 64, "float8")
    h = torchcl.to_opencl
    x = rnd(1, 4, 8, 64, dtype=torch.bfloat16)
    q, k, v = h(x[:, :4].contiguous()), h(x[:, 4:6].contiguous()), h(x[:, 6:].contiguous())
    table, pos = h(S.rope_table(64, 64)), h(torch.arange(4, dtype=torch.int32))
    slots, ptab, ctx = h(torch.arange(4, dtype=torch.int32)), h(torch.arange(8, dtype=torch.int32)[None].contiguous()), h(torch.zeros(1, dtype=torch.int32))

    def step():
        y = S.qkv_to_cache(q, k, v, None, None, table, pos, cache, slots)
        return y, cache.read(slots)[0]

    want = [torchcl.to_cpu(t) for t in step()]
    with capture_graph() as g:
        out = step()
    g.replay()
    torchcl.synchronize()
    assert all(torch.equal(torchcl.to_cpu(a), b) for a, b in zip(out, want))


# ── long calls: the forms that stream rows ─────────────────────────────────────────

@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,inter,dtype", [
    (2400, 8, 2, 128, 128, False, "bf16"), (2371, 7, 1, 96, 48, False, "f32"), (5003, 3, 3, 64, 64, True, "f16"),
    (2999, 2, 1, 256, 128, False, "bf16"), (2500, 1, 1, 512, 512, False, "f32"), (2400, 5, 3, 32, 16, False, "bf16")])
def test_qk_many_tokens(S, tokens, hq, hk, dim, rotary, inter, dtype):
    q, k, qw, kw, table, pos = qk_inputs(tokens, hq, hk, dim, rotary, dtype)
    gq, gk = rnd(8, *q.shape, dtype=q.dtype), rnd(9, *k.shape, dtype=q.dtype)
    d = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
    out = S.qk_norm_rope(*d, table.cuda(), pos.cuda(), interleaved=inter)
    got = torch.autograd.grad(out, d, [gq.cuda(), gk.cuda()])
    for x, w, g, y, dx, dw in ((q, qw, gq, out[0].detach(), got[0], got[2]), (k, kw, gk, out[1].detach(), got[1], got[3])):
        u = ROUND[x.dtype] if x.dtype != torch.float32 else 0.0
        tiny = 6e-8 if dtype == "f16" else 0.0
        want, size = ref.norm_rope(x, w, table, pos, interleaved=inter)
        within(y, want, u * want.abs() + 32 * F32 * size + tiny)
        want, dwant, size, dsize = ref.norm_rope_grad(x, w, g, table, pos, interleaved=inter)
        within(dx, want, u * want.abs() + 64 * F32 * size + tiny)
        # runs in a register, warps of a block, blocks: at most a few hundred roundings deep
        within(dw, dwant, u * dwant.abs() + 1024 * F32 * dsize)


def test_many_tokens_bad_positions_and_slots(S):
    import torchcl
    n = 2500
    q, k, qw, kw, table, pos = qk_inputs(n, 4, 2, 128, 128, "bf16")
    pos[7], pos[2000] = 5000, -3
    slots = torch.randperm(n + 100, generator=torch.Generator().manual_seed(1))[:n]
    slots[11], slots[12] = -1, 10 ** 9
    fused = torch.cat([q, k, k], 1).cuda()
    cache = S.KVCache.from_pages(*pages_for("int8", (n + 100) // 4, 2, 4, 128))
    got = S.qkv_to_cache(fused[:, :4], fused[:, 4:6], fused[:, 6:], qw.cuda(), kw.cuda(), table.cuda(), pos.cuda(), cache, slots.cuda())
    with pytest.raises(ValueError, match="out of range"):
        torchcl.synchronize()
    assert torch.isnan(got[[7, 2000]]).all() and int(torch.isnan(got).any(-1).any(-1).sum()) == 2
    keep = torch.ones(n, dtype=torch.bool)
    keep[[11, 12]] = False
    kk, v = cache.read(slots[keep].cuda(), dtype=torch.float32)
    assert torch.equal(v.cpu(), ref.stored(k[keep], "int8")[0])
    bad = torch.isnan(kk).any(-1).any(-1).cpu()
    assert torch.equal(bad, ((pos < 0) | (pos >= 5000))[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_cache_many_tokens_is_exact(S, fmt, dtype):
    n, heads, dim, size = 3001, 3, 96, 16
    k, v = rnd(1, n, heads, dim, dtype=DT[dtype], scale=7.0), rnd(2, n, heads, dim, dtype=DT[dtype], scale=1e-3)
    cache = S.KVCache.from_pages(*pages_for(fmt, n // size + 2, heads, size, dim))
    slots = torch.randperm(n, generator=torch.Generator().manual_seed(3)).cuda()
    cache.append(k.cuda(), v.cuda(), slots)
    for x, y in zip((k, v), cache.read(slots, dtype=torch.float32)):
        assert torch.equal(y.cpu(), ref.stored(x, fmt)[0])


@pytest.mark.parametrize("fmt", ["int8", "float8"])
def test_cache_quotients_are_those_of_division(S, fmt):
    """Four million quotients, steps over 60 powers of ten, ties among them: every stored
    value is that of a correctly rounded division."""
    n, dim = 32768, 128
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(n, 1, dim, generator=gen) * 10.0 ** (torch.rand(n, 1, 1, generator=gen) * 60 - 30)
    x[:, :, 64:] = (torch.randint(-254, 255, (n, 1, 64), generator=gen) * 0.5) / 127 * x.abs().amax(-1, keepdim=True)
    cache = S.KVCache.from_pages(*pages_for(fmt, n // 16, 1, 16, dim))
    slots = torch.arange(n).cuda()
    cache.append(x.cuda(), x.flip(0).cuda(), slots)
    for a, b in zip((x, x.flip(0)), cache.read(slots, dtype=torch.float32)):
        assert torch.equal(b.cpu(), ref.stored(a, fmt)[0])
