"""The serving operators beside other work: caches made on torchcl's stream and used on
torch's, caches dropped while calls run, errors of calls that still run or are replayed,
captured decoding steps, calls from two threads."""
import threading

import pytest
import torch

from test_gpu_serving import pages_for, rnd

pytestmark = pytest.mark.gpu
LONG = 200_000_000  # clocks of a wait on a stream: about a tenth of a second


@pytest.fixture(scope="module")
def S():
    from torchcl import serving
    return serving


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def busy_torchcl():
    """Work on torchcl's stream for about a tenth of a second."""
    from torchcl.runtime.context import get_queue
    with torch.cuda.stream(torch.cuda.ExternalStream(get_queue())):
        torch.cuda._sleep(LONG)


# ── one cache, two streams ───────────────────────────────────────────────────

@pytest.mark.parametrize("side", [False, True])
def test_a_new_cache_is_cleared_before_its_first_use(S, side):
    """Rows written by torch right after the constructor are there afterwards; the rest of
    8 GB is zeros."""
    x = rnd(1, 4, 8, 128, dtype=torch.bfloat16).cuda()
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    pages = 1 << 15
    slots = torch.tensor([0, 7, pages * 64 - 1, pages * 32], device="cuda")
    S.KVCache(2, 16, 8, 128, "bfloat16").append(x[:2], x[:2], slots[:2])  # (loads the kernel)
    torch.cuda.synchronize()
    busy_torchcl()
    cache = S.KVCache(pages, 64, 8, 128, "bfloat16")
    with torch.cuda.stream(stream):
        cache.append(x, -x, slots)
    torch.cuda.synchronize()
    k, v = cache.read(slots)
    assert torch.equal(k, x) and torch.equal(v, -x)
    assert not cache.read(slots - 2)[0][1:].any()


def test_pages_freed_while_torch_still_uses_them(S):
    """A cache deleted while a call on torch's stream waits to run: its pages are not those of
    the next cache, whose clearing would reach the call."""
    x = rnd(2, 64, 2, 64, dtype=torch.float16).cuda()
    slots = torch.arange(64).cuda()
    cache = S.KVCache(64, 16, 2, 64, "float16")
    cache.append(x, x, slots)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        k, v = cache.read(slots, dtype=torch.float16)
    del cache
    others = [S.KVCache(64, 16, 2, 64, "float16") for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(k, x) and torch.equal(v, x)
    assert not others[0].read(slots)[0].any()


def test_freed_pages_come_back(S):
    """Caches made, used on torch's stream and dropped in a loop do not add up."""
    from torchcl.runtime.memory import get_buffer_pool
    x = rnd(3, 4, 4, 128, dtype=torch.float16).cuda()
    used = []
    for _ in range(12):
        cache = S.KVCache(1 << 12, 64, 4, 128, "float16")
        cache.append(x, x, torch.arange(4).cuda())
        torch.cuda.synchronize()
        del cache
        used.append(get_buffer_pool().get_stats()["total_allocated_bytes"])
    assert used[-1] == used[2]


def test_torch_pages_freed_while_torchcl_still_uses_them(S):
    import torchcl
    n = 1 << 14
    x = rnd(4, n, 2, 64, dtype=torch.float16)
    cache = S.KVCache.from_pages(*pages_for("float16", n // 16, 2, 16, 64))
    cache.append(x.cuda(), x.cuda(), torch.arange(n).cuda())
    torch.cuda.synchronize()
    slots = torchcl.to_opencl(torch.arange(n).int())
    cache.read(slots, dtype=torch.float16)
    torch.full((8,), 7.0, dtype=torch.float16, device="cuda")  # (loads the kernel)
    torch.cuda.synchronize()
    busy_torchcl()
    k, _ = cache.read(slots, dtype=torch.float16)
    del cache
    waste = [torch.full((n // 16, 2, 16, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(torchcl.to_cpu(k), x)
    del waste


def test_pages_dropped_in_a_capture_go_back_after_it(S, monkeypatch):
    x = rnd(6, 1, 1, 64, dtype=torch.float16).cuda()
    cache = S.KVCache(4, 16, 1, 64, "float16")
    cache.append(x, x, torch.tensor([3], device="cuda"))
    pages = cache._pages[:2]
    with monkeypatch.context() as m:
        m.setattr(S, "_capturing", lambda: True)
        del cache
        S.KVCache(4, 16, 1, 64, "float16")
        assert not any(buf._freed for buf in pages)
    S.KVCache(4, 16, 1, 64, "float16")
    assert all(buf._freed for buf in pages)


def test_a_cache_that_does_not_fit_keeps_nothing(S):
    from torchcl import _lib as L
    from torchcl.runtime.memory import get_buffer_pool
    pool = get_buffer_pool()
    pool.empty_cache()
    before = pool.get_stats()["active_bytes"]
    pool.free(pool.allocate(12032 * 64 * 64 * 2))  # the keys' block is in the pool, the values' is not
    L.check(L.lib().ojx_pool_debug_fail_next(2))
    try:
        with pytest.raises(MemoryError):
            S.KVCache(12032, 64, 1, 64, "float16")
    finally:
        L.check(L.lib().ojx_pool_debug_fail_next(0))
    assert pool.get_stats()["active_bytes"] == before


# ── errors found on the device ───────────────────────────────────────────────

def test_errors_of_calls_that_still_run_are_reported_later(S):
    import torchcl
    x = rnd(1, 1, 1, 64).cuda()
    cache = S.KVCache.from_pages(*pages_for("int8", 2, 1, 16, 64))
    torchcl.synchronize()
    side = torch.cuda.Stream()
    bad = torch.tensor([10 ** 6], device="cuda")
    cache.append(x, x, bad - 10 ** 6)  # (loads the kernel)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        cache.append(x, x, bad)
    torchcl.synchronize()  # torchcl's stream is idle: nothing to report yet
    side.synchronize()
    with pytest.raises(ValueError, match="out of range"):
        torchcl.synchronize()
    torchcl.synchronize()  # once


def test_errors_of_replayed_calls_are_reported(S):
    import torchcl
    from torchcl.api import _get_buf
    from torchcl.jit.graph_runner import capture_graph
    from torchcl.runtime.memory import get_buffer_pool
    h = torchcl.to_opencl
    cache = S.KVCache(2, 16, 1, 64, "int8")
    x, slots = h(rnd(1, 2, 1, 64)), h(i32(3, 4))
    cache.append(x, x, slots)
    with capture_graph() as g:
        cache.append(x, x, slots)
    g.replay()
    torchcl.synchronize()
    get_buffer_pool().host_to_device(i32(3, 99), _get_buf(slots))
    for _ in range(2):
        g.replay()
        with pytest.raises(ValueError, match="out of range"):
            torchcl.synchronize()
    get_buffer_pool().host_to_device(i32(3, 5), _get_buf(slots))
    g.replay()
    torchcl.synchronize()


# ── capture and replay ───────────────────────────────────────────────────────

@pytest.mark.parametrize("tokens", [1, 5, 24])
def test_a_captured_decoding_step_with_attention(S, tokens):
    import torchcl
    from torchcl.api import _get_buf
    from torchcl.jit.graph_runner import capture_graph
    from torchcl.runtime.memory import get_buffer_pool
    h = torchcl.to_opencl
    cache = S.KVCache(16, 16, 2, 64, "float8")
    x = rnd(1, tokens, 8, 64, dtype=torch.bfloat16)
    q, k, v = h(x[:, :4].contiguous()), h(x[:, 4:6].contiguous()), h(x[:, 6:].contiguous())
    qq = h(x[:, :4].contiguous()[None])
    table, pos = h(S.rope_table(256, 64)), h(torch.arange(tokens, dtype=torch.int32) + 40)
    prompt = h(rnd(2, 100, 2, 64, dtype=torch.bfloat16))
    cache.append(prompt, prompt, h(torch.arange(100, dtype=torch.int32)))
    slots, ptab, ctx = h(torch.arange(tokens, dtype=torch.int32) + 40), h(torch.arange(16, dtype=torch.int32)[None].contiguous()), h(i32(40))

    def step():
        S.qkv_to_cache(q, k, v, None, None, table, pos, cache, slots)
        return S.tree_attention(qq, cache, ptab, ctx)

    want = torchcl.to_cpu(step())
    with capture_graph() as g:
        out = step()
    g.replay()
    torchcl.synchronize()
    assert torch.equal(torchcl.to_cpu(out), want)
    get_buffer_pool().host_to_device(i32(7), _get_buf(ctx))  # new inputs in place
    again = torchcl.to_cpu(step())
    assert not torch.equal(again, want)
    g.replay()
    torchcl.synchronize()
    assert torch.equal(torchcl.to_cpu(out), again)


# ── two threads, one stream ──────────────────────────────────────────────────

def test_two_threads_on_one_stream(S):
    """torchcl's default stream is every thread's: calls of two kernels that share a workspace,
    of two sizes, keep to themselves."""
    import torchcl
    from torchcl.serving import _qk_backward
    h = torchcl.to_opencl
    cache = S.KVCache(64, 16, 2, 64, "float16")
    x = h(rnd(1, 1024, 2, 64, dtype=torch.float16))
    cache.append(x, x, h(torch.arange(1024, dtype=torch.int32)))

    def attend(batch, tokens, seed):
        q = h(rnd(seed, batch, tokens, 8, 64, dtype=torch.float16))
        table, ctx = h(torch.arange(64, dtype=torch.int32).repeat(batch, 1)), h(torch.full((batch,), 900, dtype=torch.int32))
        return lambda: [S.tree_attention(q, cache, table, ctx)]

    def gradient(tokens, seed):
        a = [h(rnd(seed + i, tokens, n, 64)) for i, n in enumerate((4, 2, 4, 2))]
        w, table, pos = h(torch.ones(64)), h(S.rope_table(64, 64)), h(torch.arange(tokens, dtype=torch.int32) % 64)
        return lambda: _qk_backward(*a, w, w, table, pos, 1e-6, False)

    works = [[attend(1, 1, 2), gradient(40, 9)], [attend(5, 40, 5), gradient(3000, 19)]]
    want = [[[torchcl.to_cpu(t) for t in f()] for f in fs] for fs in works]
    wrong = []

    def run(fs, expected):
        try:
            kept = [[f() for f in fs] for _ in range(100)]
            for outs in kept:
                for o, e in zip(outs, expected):
                    if not all(torch.equal(torchcl.to_cpu(a), b) for a, b in zip(o, e)):
                        wrong.append("another thread's parts")
        except Exception as e:  # (a thread's exception would be lost)
            wrong.append(repr(e))

    threads = [threading.Thread(target=run, args=a) for a in zip(works, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
