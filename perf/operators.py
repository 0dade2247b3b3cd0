"""The serving operators of torchcl, measured: norms of queries and keys with the position
rotation (forward, and with its gradient), the paged cache that quantises what is written
and reads it back, attention of drafted tokens over that cache, and the verification of
drafts from given random numbers.

`run` computes a case in plain torch (elementary operations in 32 bits, one rounding at the
end) or, with `own` true, through torchcl.serving.  `exact` is each operator's definition
in 64 bits.
"""
import math
import pathlib
import random
import sys

import torch

own = False

_PACKAGE = str(pathlib.Path(__file__).resolve().parents[1] / "ojasx-open-source-cuda-_b200")
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2, "int8": 1, "float8": 1}
_TOP = {"int8": 127.0, "float8": 448.0}  # largest magnitude each quantised format holds
_UNITS = float(1 << 38)                  # verification counts probability in units of 2^-38
_THETA = 500000.0


def _serving():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from torchcl import serving
    return serving


# ── the cases ────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decoding step of eight sequences: a few rows, where only latency counts
        dict(name="qk_token", op="qk", tokens=8, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, dtype="bf16", train=False),
        # a training step's 16k tokens, forward and gradients
        dict(name="qk_train", op="qk", tokens=16384, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, dtype="bf16", train=True),
        # a small model in float32: odd token count, one shared key head, half of each head rotated
        dict(name="qk_train_odd_f32", op="qk", tokens=1537, q_heads=7, kv_heads=1, head_dim=96,
             rotary=48, interleaved=True, dtype="f32", train=True),
        # a prompt chunk after its fused projection: q, k, v are slices of one tensor; k is
        # normed, rotated and quantised into the cache with v in the same pass
        dict(name="prompt_to_cache_int8", op="qkv", tokens=8192, q_heads=32, kv_heads=8, head_dim=128,
             rotary=128, interleaved=False, dtype="bf16", format="int8", page=64),
        # one new token of each of 64 sequences written to a float8 cache and read back
        dict(name="cache_tokens_float8", op="cache", tokens=64, kv_heads=8, head_dim=128, dtype="f16",
             format="float8", page=16),
        # long prompts moved into an int8 cache and read back, float32 source
        dict(name="cache_prompt_int8", op="cache", tokens=50021, kv_heads=4, head_dim=128, dtype="f32",
             format="int8", page=128),
        # the latency of one sequence's next token over a short cache
        dict(name="attend_one_short", op="attend", batch=1, tokens=1, context=701, q_heads=32, kv_heads=8,
             head_dim=128, dtype="bf16", format="bf16", page=16, ragged=False, tree=False),
        # a decoding batch over a quantised cache, contexts of very different lengths
        dict(name="attend_batch_int8", op="attend", batch=64, tokens=1, context=8191, q_heads=32, kv_heads=8,
             head_dim=128, dtype="bf16", format="int8", page=64, ragged=False, tree=False),
        # verification pass of draft trees, 48 nodes for each of eight sequences
        dict(name="attend_tree_float8", op="attend", batch=8, tokens=48, context=16000, q_heads=32, kv_heads=8,
             head_dim=128, dtype="f16", format="float8", page=32, ragged=True, tree=True),
        # two very long contexts, a small tree, wide sharing of key heads
        dict(name="attend_tree_long", op="attend", batch=2, tokens=16, context=131000, q_heads=32, kv_heads=4,
             head_dim=128, dtype="bf16", format="bf16", page=64, ragged=False, tree=True),
        # chains of sampled drafts, the rejection form with the draft's own probabilities
        dict(name="verify_chain", op="verify", batch=4, tokens=6, vocab=32000, dtype="f32", sampled=True,
             chain=True),
        # trees of the draft's likeliest tokens for a full batch
        dict(name="verify_tree", op="verify", batch=64, tokens=48, vocab=131072, dtype="f32", sampled=False,
             chain=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    op = rng.choice(["qk", "qkv", "cache", "attend", "attend", "verify"])
    if op in ("qk", "qkv"):
        head_dim = rng.choice([64, 96, 128, 256])
        kv = rng.choice([1, 2, 3, 4, 8])
        q = kv * rng.choice([1, 2, 4, 5, 7, 8])
        most = min(16384, 16384 * 40 * 128 // ((q + kv) * head_dim))
        case = dict(op=op, tokens=_log(rng, 1, most), q_heads=q, kv_heads=kv, head_dim=head_dim,
                    rotary=rng.choice([head_dim, head_dim // 2]), interleaved=rng.random() < 0.3)
        if op == "qk":
            return dict(case, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]) if most < 8192 else rng.choice(["bf16", "f16"]),
                        train=rng.random() < 0.6)
        return dict(case, dtype=rng.choice(["bf16", "f16"]), format=rng.choice(["bf16", "f16", "int8", "float8"]),
                    page=rng.choice([16, 32, 64, 128]))
    if op == "cache":
        heads, head_dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 96, 128, 256])
        most = 50000 * 4 * 128 // (heads * head_dim)
        return dict(op=op, tokens=_log(rng, 1, most), kv_heads=heads, head_dim=head_dim,
                    dtype=rng.choice(["f32", "bf16", "f16"]), format=rng.choice(["bf16", "f16", "int8", "float8"]),
                    page=rng.choice([16, 32, 64, 128]))
    if op == "attend":
        dtype = rng.choice(["bf16", "f16"])
        fmt = rng.choice([dtype, "int8", "float8"])
        kv, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        group = rng.choice([1, 2, 4, 5, 7, 8])
        batch, tokens = _log(rng, 1, 64), _log(rng, 1, 64)
        # at most the listed cases' bytes and multiplications
        most = min(131000, 250e6 / (batch * kv * head_dim * _SIZES[fmt]), 25e9 / (batch * tokens * group * kv * head_dim))
        return dict(op=op, batch=batch, tokens=tokens, context=_log(rng, 1, max(2, most)), q_heads=kv * group,
                    kv_heads=kv, head_dim=head_dim, dtype=dtype, format=fmt, page=rng.choice([16, 32, 64, 128]),
                    ragged=rng.random() < 0.5, tree=rng.random() < 0.7)
    vocab = _log(rng, 1000, 131072)
    tokens = _log(rng, 1, 64)
    sampled = rng.random() < 0.5
    most = max(1, min(64, int(200e6 / (vocab * tokens))))
    return dict(op="verify", batch=_log(rng, 1, most), tokens=tokens, vocab=vocab,
                dtype=rng.choice(["f32", "f32", "bf16"]), sampled=sampled, chain=rng.random() < 0.4)


def work(case):
    c = case
    op = c["op"]
    if op in ("qk", "qkv"):
        rows = c["tokens"] * (c["q_heads"] + c["kv_heads"])
        elems = rows * c["head_dim"]
        size = _SIZES[c["dtype"]]
        side = c["tokens"] * (8 + 4 * c["rotary"])  # positions and their rotations
        if op == "qk":
            return {"bytes": elems * size * (4 if c["train"] else 2) + side, "flops": elems * (22 if c["train"] else 7)}
        kv = c["tokens"] * c["kv_heads"] * c["head_dim"]
        cached = 2 * kv * _SIZES[c["format"]] + (8 * c["tokens"] * c["kv_heads"] if c["format"] in _TOP else 0)
        return {"bytes": elems * size + kv * size + (elems - kv) * size + cached + 2 * kv * size + side, "flops": elems * 8}
    if op == "cache":
        kv = 2 * c["tokens"] * c["kv_heads"] * c["head_dim"]
        scales = 8 * c["tokens"] * c["kv_heads"] if c["format"] in _TOP else 0
        return {"bytes": kv * (2 * _SIZES[c["dtype"]] + _SIZES[c["format"]]) + scales + 8 * c["tokens"], "flops": 3 * kv}
    if op == "attend":
        keys = sum(ctx + t for ctx, t in zip(_contexts(c), _drafts(c)))
        pairs = sum((ctx + t) * t for ctx, t in zip(_contexts(c), _drafts(c)))
        row = c["kv_heads"] * (c["head_dim"] * _SIZES[c["format"]] + (4 if c["format"] in _TOP else 0))
        io = 2 * c["batch"] * c["tokens"] * c["q_heads"] * c["head_dim"] * 2
        return {"bytes": 2 * keys * row + io, "flops": 4 * pairs * c["q_heads"] * c["head_dim"]}
    rows = 2 if c["sampled"] else 1  # the row that the next token is drawn from, and its draft's
    return {"bytes": c["batch"] * (c["vocab"] * rows * _SIZES[c["dtype"]] + c["tokens"] * 32), "flops": c["batch"] * c["vocab"] * 4 * rows}


def _contexts(c):
    """Each sequence's tokens in the cache: from all of `context` down to a third of it."""
    n = c["batch"]
    return [max(0, c["context"] - (c["context"] * 2 * b) // (3 * n)) for b in range(n)]


def _drafts(c):
    return [max(1, c["tokens"] - b % 3) if c["ragged"] else c["tokens"] for b in range(c["batch"])]


# ── inputs ───────────────────────────────────────────────────────────────────

def _quantised(x, fmt):
    """Values as a cache of this format holds them: (stored, scale or None)."""
    if fmt not in _TOP:
        return x.to(_DTYPES[fmt]), None
    scale = x.float().abs().amax(-1) / _TOP[fmt]
    q = x.float() / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    if fmt == "int8":
        return torch.round(q).clamp(-127, 127).to(torch.int8), scale
    return q.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _parents(rng, tokens, chain):
    """A tree's parents: node 0 is the root; drafts hang on recent nodes, several to one."""
    return [-1] + [i - 1 if chain else rng.randrange(max(0, i - 9), i) for i in range(1, tokens)]


def _ancestor_words(parents):
    """Bit j of row i: node j is i or an ancestor of i (int64 words of 64 nodes)."""
    sees = []
    for i, p in enumerate(parents):
        sees.append((sees[p] if p >= 0 else 0) | (1 << i))
    words = (len(parents) + 63) // 64
    signed = lambda w: w - (1 << 64) if w >> 63 else w  # noqa: E731
    return [[signed((s >> (64 * w)) & ((1 << 64) - 1)) for w in range(words)] for s in sees]


def _empty_cache(pages, heads, page, head_dim, fmt, dev):
    dtype = {"int8": torch.int8, "float8": torch.float8_e4m3fn}.get(fmt) or _DTYPES[fmt]
    shape = (pages, heads, page, head_dim)
    data = [torch.zeros(shape, dtype=torch.uint8 if fmt in _TOP else dtype, device=dev).view(dtype) for _ in "kv"]
    scales = [torch.zeros(shape[:3], device=dev) if fmt in _TOP else None for _ in "kv"]
    return data + scales


def prepare(case, seed):
    c, dev = case, "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    s = dict(case=c)
    if c["op"] in ("qk", "qkv"):
        n, hq, hk, d = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
        dtype = _DTYPES[c["dtype"]]
        span = 32768
        freq = _THETA ** (-torch.arange(0, c["rotary"], 2, dtype=torch.float64) / c["rotary"])
        angle = torch.arange(span, dtype=torch.float64)[:, None] * freq
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float().to(dev)
        s["positions"] = (torch.arange(n, device=dev) + rng.randrange(span)) % span
        s["weights"] = [(1 + 0.2 * randn(d)).to(dtype) for _ in "qk"]
        heads = hq + hk + (hk if c["op"] == "qkv" else 0)
        x = (randn(n, heads, d) * (0.5 + 2 * torch.rand(heads, 1, generator=gen, device=dev))).to(dtype)
        if c["op"] == "qk":
            s["q"], s["k"] = x[:, :hq].contiguous(), x[:, hq:].contiguous()
            if c["train"]:
                s["grads"] = [randn(*t.shape).to(dtype) for t in (s["q"], s["k"])]
                for t in (s["q"], s["k"], *s["weights"]):
                    t.requires_grad_(True)
        else:
            s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if c["op"] == "cache":
        shape, dtype = (c["tokens"], c["kv_heads"], c["head_dim"]), _DTYPES[c["dtype"]]
        s["k"], s["v"] = [(randn(*shape) * (0.25 + 3 * torch.rand(shape[2], generator=gen, device=dev))).to(dtype) for _ in "kv"]
    if c["op"] in ("qkv", "cache"):
        pages = (c["tokens"] + c["page"] - 1) // c["page"] + 3
        s["pages"] = _empty_cache(pages, c["kv_heads"], c["page"], c["head_dim"], c["format"], dev)
        at = torch.arange(c["tokens"], device=dev) + rng.randrange(c["page"])
        order = torch.randperm(pages, generator=gen, device=dev)
        s["slots"] = order[at // c["page"]] * c["page"] + at % c["page"]
    if c["op"] == "attend":
        b, t, d = c["batch"], c["tokens"], c["head_dim"]
        contexts, drafts = _contexts(c), _drafts(c)
        width = (max(x + t for x in contexts) + c["page"] - 1) // c["page"]
        s["pages"] = _empty_cache(b * width, c["kv_heads"], c["page"], d, c["format"], dev)
        tilt = 0.3 + torch.rand(c["kv_heads"], 1, d, generator=gen, device=dev)
        for first in range(0, b * width, 256):  # filled in parts: the float32 values are large
            part = slice(first, min(first + 256, b * width))
            for i in range(2):
                x = randn(part.stop - part.start, c["kv_heads"], c["page"], d) * tilt
                data, scale = _quantised(x, c["format"])
                s["pages"][i][part] = data
                if scale is not None:
                    s["pages"][2 + i][part] = scale
        s["page_table"] = torch.randperm(b * width, generator=gen, device=dev).reshape(b, width).int()
        s["contexts"] = torch.tensor(contexts, dtype=torch.int32, device=dev)
        s["drafts"] = torch.tensor(drafts, dtype=torch.int32, device=dev)
        words = [_ancestor_words(_parents(rng, t, not c["tree"])) for _ in range(b)]
        s["mask"] = torch.tensor(words, dtype=torch.int64, device=dev)
        s["q"] = (1.5 * randn(b, t, c["q_heads"], d)).to(_DTYPES[c["dtype"]])
        s["width"] = width
    if c["op"] == "verify":
        b, t, v = c["batch"], c["tokens"], c["vocab"]
        parents = [_parents(rng, t, c["chain"]) for _ in range(b)]
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device=dev)
        s["uniforms"] = torch.rand(b, t, generator=gen, device=dev)
        target = torch.empty(b, t, v, dtype=_DTYPES[c["dtype"]], device=dev)
        draft = torch.empty_like(target) if c["sampled"] else None
        tokens = torch.zeros(b, t, dtype=torch.int64, device=dev)
        index = s["parents"].long().clamp(min=0)
        for i in range(b):
            logits = 2.5 * randn(t, v)
            target[i] = torch.softmax(logits, -1).to(target.dtype)
            guess = torch.softmax(logits + 0.7 * randn(t, v), -1)
            if c["sampled"]:  # each draft drawn from its parent's draft distribution
                draft[i] = guess.to(target.dtype)
                tokens[i] = torch.multinomial(guess[index[i]], 1, generator=gen)[:, 0]
            else:             # the k-th child of a node is its draft's k-th likeliest token
                best = guess.topk(min(t, v), -1).indices
                kth = [parents[i][:j].count(parents[i][j]) for j in range(t)]
                tokens[i] = best[index[i], torch.tensor(kth, device=dev)]
        s.update(target=target, draft=draft, tokens=tokens.int())
    if own and "pages" in s:
        s["cache"] = _serving().KVCache.from_pages(*s["pages"])
    return s


# ── the plain forms ──────────────────────────────────────────────────────────

def _rotate(x, table, positions, rotary, interleaved):
    half = rotary // 2
    row = table[positions.long()]
    cos, sin = row[:, None, :half], row[:, None, half:]
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rotary]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _norm_rotate(x, weight, s):
    c = s["case"]
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    return _rotate(y, s["table"], s["positions"], c["rotary"], c["interleaved"])


def _stored(x, fmt):
    data, scale = _quantised(x, fmt)
    return data.float() if scale is None else data.float() * scale[..., None]


def _write(s, k, v):
    """k and v into the pages at their slots, and what a reader gets back."""
    c = s["case"]
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    back = []
    for i, x in enumerate((k, v)):
        data, scale = _quantised(x, c["format"])
        pages = s["pages"][i]
        if scale is None:
            pages[page, :, at] = data
            back.append(pages[page, :, at].float())
        else:  # 8-bit values move as bytes
            pages.view(torch.uint8)[page, :, at] = data.view(torch.uint8)
            s["pages"][2 + i][page, :, at] = scale
            got = pages.view(torch.uint8)[page, :, at].view(data.dtype).float()
            back.append(got * s["pages"][2 + i][page, :, at][..., None])
    return [x.to(_DTYPES[c["dtype"]]) for x in back]


def _plain_attend(s):
    c = s["case"]
    b, t, hq, d = s["q"].shape
    hk = c["kv_heads"]
    keys = s["width"] * c["page"]

    def dense(i):
        table = s["page_table"].long()
        if c["format"] in _TOP:
            x = s["pages"][i].view(torch.uint8)[table].view(s["pages"][i].dtype).float()
            x = x * s["pages"][2 + i][table][..., None]
        else:
            x = s["pages"][i][table].float()
        return x.permute(0, 2, 1, 3, 4).reshape(b, hk, keys, d)

    col = torch.arange(keys, device="cuda")
    back = col[None] - s["contexts"][:, None]                       # < 0: context, else draft
    bits = (s["mask"][:, :, :, None] >> torch.arange(64, device="cuda")) & 1
    tree = bits.reshape(b, t, -1)[:, :, :t].bool()
    tree = tree & (torch.arange(t, device="cuda") < s["drafts"][:, None])[:, None]
    seen = torch.gather(tree, 2, back.clamp(0, t - 1)[:, None].expand(b, t, keys)) & (back < t)[:, None]
    seen = (seen | (back < 0)[:, None]) & (torch.arange(t, device="cuda") < s["drafts"][:, None])[:, :, None]
    q = s["q"].float().permute(0, 2, 1, 3).reshape(b, hk, hq // hk, t, d)
    score = torch.matmul(q.reshape(b, hk, -1, d), dense(0).transpose(2, 3)) * d ** -0.5
    score = score.reshape(b, hk, hq // hk, t, keys).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(b, hk, -1, keys), dense(1)).reshape(b, hk, hq // hk, t, d)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.reshape(b, hq, t, d).permute(0, 2, 1, 3).to(s["q"].dtype)


def _units(x):
    return torch.floor(x * _UNITS).to(torch.int64)


def _plain_verify(s):
    target, draft, tokens, parents, u = s["target"], s["draft"], s["tokens"].long(), s["parents"], s["uniforms"]
    b, t, v = target.shape
    row = torch.arange(b, device="cuda")
    clean = lambda p: torch.nan_to_num(p.float(), nan=0.0).clamp(0, 1)  # noqa: E731
    at = torch.zeros(b, dtype=torch.int64, device="cuda")               # the node reached
    left, mass = clean(target[row, at]), torch.ones(b, device="cuda")   # what is left of its row
    path = torch.full((b, t), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    count = torch.zeros(b, dtype=torch.int32, device="cuda")
    for i in range(1, t):  # a node is tried when its parent is the one reached
        x = tokens[:, i]
        tried = parents[:, i] == at
        chance = clean(draft[row, at, x]) if draft is not None else torch.ones(b, device="cuda")
        yes = tried & (u[:, i] * (chance * mass) < left[row, x])
        no = tried & ~yes
        if draft is not None:
            rest = (left - mass[:, None] * clean(draft[row, at])).clamp(min=0)
            rest_mass = (_units(rest).sum(1).double() / _UNITS).float()
        else:
            rest_mass = (mass - left[row, x]).clamp(min=0)
            rest = left.clone()
            rest[row, x] = 0.0
        at = torch.where(yes, i, at)
        count = count + yes.int()
        path[row, torch.where(yes, count.long(), 0)] = torch.where(yes, i, 0).int()
        left = torch.where(yes[:, None], clean(target[row, at]), torch.where(no[:, None], rest, left))
        mass = torch.where(yes, torch.ones_like(mass), torch.where(no, rest_mass, mass))
    weight = _units(left)
    empty = weight.sum(1) == 0
    weight = torch.where(empty[:, None], _units(clean(target[row, at])), weight)
    total = weight.sum(1)
    u24 = torch.floor(u[:, 0] * (1 << 24)).to(torch.int64).clamp(0, (1 << 24) - 1)
    goal = u24 * (total >> 24) + ((u24 * (total & ((1 << 24) - 1))) >> 24)
    token = (weight.cumsum(1) <= goal[:, None]).sum(1)
    return path, count, torch.where(total > 0, token, -1).int()


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "qk":
        q, k = [_norm_rotate(s[n], w, s).to(s[n].dtype) for n, w in zip("qk", s["weights"])]
        if not c["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"], *s["weights"]], s["grads"]))
    if c["op"] == "qkv":
        q = _norm_rotate(s["q"], s["weights"][0], s).to(s["q"].dtype)
        return q, *_write(s, _norm_rotate(s["k"], s["weights"][1], s), s["v"])
    if c["op"] == "cache":
        return _write(s, s["k"], s["v"])
    return _plain_attend(s) if c["op"] == "attend" else _plain_verify(s)


def _run_own(s, c):
    serving = _serving()
    if c["op"] == "qk":
        q, k = serving.qk_norm_rope(s["q"], s["k"], *s["weights"], s["table"], s["positions"], interleaved=c["interleaved"])
        if not c["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"], *s["weights"]], s["grads"]))
    if c["op"] == "qkv":
        q = serving.qkv_to_cache(s["q"], s["k"], s["v"], *s["weights"], s["table"], s["positions"], s["cache"], s["slots"],
                                 interleaved=c["interleaved"])
        return q, *s["cache"].read(s["slots"], dtype=s["q"].dtype)
    if c["op"] == "cache":
        s["cache"].append(s["k"], s["v"], s["slots"])
        return s["cache"].read(s["slots"], dtype=s["k"].dtype)
    if c["op"] == "attend":
        return serving.tree_attention(s["q"], s["cache"], s["page_table"], s["contexts"], mask=s["mask"], draft_lens=s["drafts"])
    return serving.verify_drafts(s["target"], s["tokens"], s["parents"], s["uniforms"], draft_probs=s["draft"])


# ── the definitions in 64 bits ───────────────────────────────────────────────

def _exact_qk(x, w, g, cos, sin, c):
    """The normed and rotated rows, and with g the gradients of x and w."""
    r, d = c["rotary"], c["head_dim"]
    first = torch.arange(0, r, 2) if c["interleaved"] else torch.arange(r // 2)
    second = first + (1 if c["interleaved"] else r // 2)
    turn = torch.eye(d, dtype=torch.float64, device=x.device).expand(x.shape[0], d, d).clone()  # y = turn @ normed
    turn[:, first, first], turn[:, second, second] = cos, cos
    turn[:, first, second], turn[:, second, first] = -sin, sin
    x, w = x.double(), w.double()
    inverse = (x.pow(2).sum(-1, keepdim=True) / d + 1e-6).pow(-0.5)
    y = torch.einsum("nij,nhj->nhi", turn, x * inverse * w)
    if g is None:
        return y, None, None
    back = torch.einsum("nij,nhi->nhj", turn, g.double())
    inner = (back * w * x).sum(-1, keepdim=True)
    return y, inverse * back * w - x * inverse.pow(3) * inner / d, (back * x * inverse).sum((0, 1))


def _exact_rows(x, fmt):
    """What a cache of this format stands for after x was written, in 64 bits."""
    if fmt not in _TOP:
        return x.to(_DTYPES[fmt]).double()
    step = x.double().abs().amax(-1, keepdim=True) / _TOP[fmt]
    level = x.double() / step.clamp(min=1e-300)
    if fmt == "float8":  # three fraction bits; below 2^-6 the spacing stays 2^-9
        spacing = torch.exp2(torch.floor(torch.log2(level.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(level / spacing) * spacing * step
    return torch.round(level) * step


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "verify":
        return None
    if c["op"] in ("qk", "qkv"):
        outs = []
        heads = dict(q=s["weights"][0], k=s["weights"][1])
        for i, n in enumerate("qk"):
            w = heads[n].detach()
            y, dx, dw = [], [], 0
            for at in range(0, c["tokens"], 2048):
                part = slice(at, at + 2048)
                row = s["table"][s["positions"][part]].double()
                g = s["grads"][i][part] if c.get("train") else None
                got = _exact_qk(s[n].detach()[part], w, g, row[:, :c["rotary"] // 2], row[:, c["rotary"] // 2:], c)
                y.append(got[0])
                if g is not None:
                    dx.append(got[1])
                    dw = dw + got[2]
            outs.append((torch.cat(y), torch.cat(dx) if dx else None, dw))
        (q, dq, dqw), (k, dk, dkw) = outs
        if c["op"] == "qkv":
            return q, _exact_rows(k, c["format"]), _exact_rows(s["v"], c["format"])
        return (q, k, dq, dk, dqw, dkw) if c["train"] else (q, k)
    if c["op"] == "cache":
        return [_exact_rows(s[n], c["format"]) for n in "kv"]
    outs = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = c["q_heads"] // c["kv_heads"]
    for b, (ctx, t) in enumerate(zip(_contexts(c), _drafts(c))):
        at = torch.arange(ctx + t, device="cuda")
        page = s["page_table"][b].long()[at // c["page"]]
        sees = torch.ones(t, ctx + t, dtype=torch.bool, device="cuda")
        words = s["mask"][b].tolist()
        tree = [[bool((words[i][j // 64] >> (j % 64)) & 1) for j in range(t)] for i in range(t)]
        sees[:, ctx:] = torch.tensor(tree, device="cuda")
        for h in range(c["kv_heads"]):
            k, v = [p[page, h, at % c["page"]] if c["format"] not in _TOP
                    else p.view(torch.uint8)[page, h, at % c["page"]].view(p.dtype) for p in s["pages"][:2]]
            k, v = k.double(), v.double()
            if c["format"] in _TOP:
                k, v = [x * sc[page, h, at % c["page"]].double()[:, None] for x, sc in zip((k, v), s["pages"][2:])]
            q = s["q"][b, :t, h * group:(h + 1) * group].double().transpose(0, 1)
            score = (q @ k.T) / math.sqrt(c["head_dim"])
            outs[b, :t, h * group:(h + 1) * group] = (torch.softmax(score.masked_fill(~sees, -math.inf), -1) @ v).transpose(0, 1)
    return outs
