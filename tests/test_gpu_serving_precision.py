"""Bits of tree_attention's weights, for every kernel (rows a key head) and cache format:
few keys whose values cancel, long contexts under one large score, values of any size.

Tolerances, in units of size = sum of weight * |value|: a weight is rounded once to f16 (half
a spacing: 2^-11) or, over bf16 values, held in two bf16 numbers (2^-17); its score's float32
errors and the exponential add less than 2^-15.  One rounding of the output joins them."""
import pytest
import torch

import serving_reference as ref
from serving_reference import ROUND
from test_gpu_serving import DT, pages_for, rnd, within

pytestmark = pytest.mark.gpu
ROWS = [(2, 4), (4, 4), (20, 4), (40, 4)]  # tokens, query heads of one key head: every kernel


@pytest.fixture(scope="module")
def S():
    from torchcl import serving
    return serving


def weight_bits(fmt):
    return 2.0 ** -17 + 2.0 ** -15 if fmt == "bfloat16" else 2.0 ** -11 + 2.0 ** -15


def over_context(S, q, k, v, fmt, size=16, batch=1):
    """tree_attention of q [tokens, heads, dim] over the keys alone (no draft is visible)."""
    n, hk, dim = k.shape
    t = q.shape[0]
    pages = (n + t + size - 1) // size
    cache = S.KVCache.from_pages(*pages_for(fmt, pages, hk, size, dim))
    cache.append(k.cuda(), v.cuda(), torch.arange(n).cuda())
    table = torch.arange(pages).int().repeat(batch, 1).cuda()
    return S.tree_attention(q[None].repeat(batch, 1, 1, 1).cuda(), cache, table, torch.full((batch,), n, dtype=torch.int32).cuda(),
                            mask=torch.zeros(t, (t + 63) // 64, dtype=torch.int64).cuda())


CACHES = [("bf16", "bfloat16"), ("f16", "float16"), ("f16", "int8"), ("f16", "float8"), ("bf16", "int8"), ("bf16", "float8")]


@pytest.mark.parametrize("dtype,fmt", CACHES)
@pytest.mark.parametrize("t,hq", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
def test_few_keys_that_cancel(S, dtype, fmt, t, hq, dim):
    k, v = rnd(1, 6, 1, dim, dtype=DT[dtype]), rnd(2, 6, 1, dim, dtype=DT[dtype])
    v[1::2] = -v[::2]
    q = rnd(3, t, hq, dim, dtype=DT[dtype], scale=0.5)
    got = over_context(S, q, k, v, fmt)[0]
    want, size = ref.attend(q, ref.stored(k, fmt)[0], ref.stored(v, fmt)[0], torch.ones(t, 6, dtype=torch.bool), dim ** -0.5)
    within(got, want, ROUND[got.dtype] * want.abs() + weight_bits(fmt) * size + 6e-8)


@pytest.mark.parametrize("fmt", ["bfloat16", "float16", "int8", "float8"])
@pytest.mark.parametrize("t,hq", ROWS)
@pytest.mark.parametrize("step_ratio,sink", [(1, 1.0), (1, -0.0625), (4, 1.0), (4, -0.0625), (64, 1.0), (64, -0.0625), (256, 1.0)])
def test_long_context_under_large_scores(S, fmt, t, hq, step_ratio, sink):
    """65536 keys of one weight under twelve whose weights are 2^16.3 times that, a value of
    `step_ratio` and next to no weight in every block of 32: the many carry a sixteenth of
    the output.  As many sequences as SMs, so that one CTA takes a whole one."""
    dtype = "bf16" if fmt == "bfloat16" else "f16"
    n, dim = 65536, 64
    k, v = torch.zeros(n, 1, dim), torch.ones(n, 1, dim)
    k[:, 0, 0] = 1.0
    k[5::32, 0, 0] = -40.0
    v[5::32] = step_ratio
    k[:384:32, 0, 0] = 12.3
    v[:384:32] = sink
    k, v = k.to(DT[dtype]), v.to(DT[dtype])
    q = torch.zeros(t, hq, dim, dtype=DT[dtype])
    q[..., 0] = 8.0
    got = over_context(S, q, k, v, fmt, size=64, batch=148)
    want, size = ref.attend(q[:1, :1], ref.stored(k, fmt)[0], ref.stored(v, fmt)[0], torch.ones(1, n, dtype=torch.bool), dim ** -0.5)
    want, size = (x.expand(148, t, hq, dim) for x in (want, size))
    within(got, want, ROUND[got.dtype] * want.abs() + weight_bits(fmt) * size)


@pytest.mark.parametrize("fmt", ["int8", "float8"])
@pytest.mark.parametrize("t,hq", ROWS)
@pytest.mark.parametrize("scale", [1e-26, 1e-18, 1.0, 1e18, 1e30, 3e34])
def test_values_of_any_size(S, fmt, t, hq, scale):
    """One step a row: values far from one, and among them rows of a tenth or no size."""
    dim, n = 64, 40
    k, v = rnd(1, n, 1, dim, dtype=torch.bfloat16), rnd(2, n, 1, dim) * scale
    v[::3] *= 0.1
    v[7] = 0.0
    v = v.bfloat16()
    q = rnd(3, t, hq, dim, dtype=torch.bfloat16)
    got = over_context(S, q, k, v, fmt)[0]
    want, size = ref.attend(q, ref.stored(k, fmt)[0], ref.stored(v, fmt)[0], torch.ones(t, n, dtype=torch.bool), dim ** -0.5)
    within(got, want, ROUND[got.dtype] * want.abs() + weight_bits(fmt) * size)


@pytest.mark.parametrize("dtype,fmt", CACHES)
@pytest.mark.parametrize("t,hq", ROWS)
def test_the_same_call_gives_the_same_bits(S, dtype, fmt, t, hq):
    """Parts of a sequence are joined in a fixed order."""
    n = 20000
    k, v, q = rnd(1, n, 1, 64, dtype=DT[dtype]), rnd(2, n, 1, 64, dtype=DT[dtype]), rnd(3, t, hq, 64, dtype=DT[dtype], scale=2.0)
    cache = S.KVCache.from_pages(*pages_for(fmt, n // 64 + 2, 1, 64, 64))
    cache.append(k.cuda(), v.cuda(), torch.arange(n).cuda())
    args = (q[None].cuda(), cache, torch.arange(n // 64 + 2).int()[None].cuda(), torch.tensor([n - t], dtype=torch.int32).cuda())
    first = S.tree_attention(*args)
    assert all(torch.equal(S.tree_attention(*args), first) for _ in range(8))
