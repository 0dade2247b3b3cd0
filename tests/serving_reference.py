"""Plain 64-bit implementations of the serving operators, on the CPU, for their tests."""
from __future__ import annotations

import math

import numpy as np
import torch

# half of the spacing of neighbouring values, relative: the error of one rounding
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TOP = {"int8": 127.0, "float8": 448.0}


def pairs(dim, rotary, interleaved):
    i = torch.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def turn(x, table, positions, interleaved, sign=1.0):
    """Rows x [tokens, heads, dim] (64-bit) turned by their tokens' angles."""
    rotary = table.shape[1]
    a, b = pairs(x.shape[-1], rotary, interleaved)
    row = table.double()[positions.long()][:, None]
    cos, sin = row[..., :rotary // 2], sign * row[..., rotary // 2:]
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def norm_rope(x, weight, table, positions, eps=1e-6, interleaved=False):
    """(turned rows, |normed a| + |normed b| of each element's pair)."""
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    n = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    a, b = pairs(x.shape[-1], table.shape[1], interleaved)
    size = n.abs()
    both = size[..., a] + size[..., b]
    size[..., a], size[..., b] = both, both.clone()
    return turn(n, table, positions, interleaved), size


def norm_rope_grad(x, weight, g, table, positions, eps=1e-6, interleaved=False):
    """(dx, dw) by the formula, and a size for each element that bounds its rounding."""
    x, g = x.double(), g.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    back = turn(g, table, positions, interleaved, -1.0)
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    h = back * w
    inner = (h * x).mean(-1, keepdim=True)
    dx = r * h - x * r.pow(3) * inner
    norm = g.norm(dim=-1, keepdim=True) * w.abs().max()
    size = r * norm * (1 + x.abs() * r)
    terms = back * x * r
    return dx, terms.sum((0, 1)), size, (g.norm(dim=-1, keepdim=True) * (x.abs() * r)).sum((0, 1))


def stored(x, fmt):
    """(what a cache of this format reads back after x was written, in float32; the steps)."""
    x = x.float()
    if fmt not in TOP:
        return x.to(getattr(torch, fmt)).float(), None
    step = x.abs().amax(-1, keepdim=True) * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32)
    fine = (step > 0) & torch.isfinite(step)
    q = x / torch.where(fine, step, torch.ones_like(step))
    if fmt == "int8":
        q = torch.round(q).clamp(-127, 127)
    else:
        q = q.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    q = torch.where(fine, q, torch.zeros_like(q))
    return q * step, step[..., 0]


def attend(q, k, v, visible, scale):
    """One sequence: q [t, hq, d], k and v [keys, hk, d] (64-bit), visible [t, keys].
    (out, sum of weight * |v|): hidden keys take no part, whatever they hold."""
    t, hq, d = q.shape
    group = hq // k.shape[1]
    out, size = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, d, dtype=torch.float64)
    for i in range(t):
        see = visible[i].nonzero()[:, 0]
        if not len(see):
            continue
        for h in range(hq):
            kk, vv = k[see, h // group].double(), v[see, h // group].double()
            p = torch.softmax(kk @ q[i, h].double() * scale, 0)
            out[i, h], size[i, h] = p @ vv, p @ vv.abs()
    return out, size


def words_to_bool(words, tokens):
    """[tokens, words] int64 -> [tokens, tokens] bool"""
    w = words.numpy().astype(np.int64).view(np.uint64)
    return torch.tensor([[bool((int(w[i, j // 64]) >> (j % 64)) & 1) for j in range(tokens)] for i in range(tokens)])


def verify(target, tokens, parents, uniforms, draft):
    """One sequence, node by node.  float32 where the definition says so, whole numbers else."""
    f = np.float32
    clean = lambda p: np.minimum(np.maximum(np.nan_to_num(p.astype(f), nan=0.0), f(0)), f(1))  # noqa: E731
    units = lambda r: [int(x) for x in np.floor(r.astype(np.float64) * 2.0 ** 38)]  # noqa: E731
    node, path, left, mass = 0, [0], clean(target[0]), f(1)
    for i in range(1, len(tokens)):
        if tokens[i] < 0 or parents[i] != node:
            continue
        x = tokens[i]
        chance = clean(draft[node])[x] if draft is not None else f(1)
        if f(uniforms[i] * f(chance * mass)) < left[x]:
            node, left, mass = i, clean(target[i]), f(1)
            path.append(i)
        elif draft is not None:
            left = np.maximum(left - mass * clean(draft[node]), f(0)).astype(f)
            mass = f(float(sum(units(left))) / 2.0 ** 38)
        else:
            mass = max(f(mass - left[x]), f(0))
            left = left.copy()
            left[x] = 0
    w = units(left)
    if sum(w) == 0:
        w = units(clean(target[node]))
    total = sum(w)
    if total == 0:
        return path, -1
    goal = (min(max(math.floor(f(uniforms[0] * f(1 << 24))), 0), (1 << 24) - 1) * total) >> 24
    run = 0
    for v, x in enumerate(w):
        run += x
        if run > goal:
            return path, v
