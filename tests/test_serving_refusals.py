"""What the serving operators refuse before any device work: caches of another device,
addresses that a kernel could not write, arithmetic on index handles."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from torchcl import _lib as L
from torchcl import serving


def bare_cache(device, pooled=False):
    """A KVCache without pages, as if made on `device`."""
    cache = serving.KVCache.__new__(serving.KVCache)
    cache._owned, cache._pooled, cache._shared, cache._pages, cache._device = False, pooled, False, [], device
    cache._desc, cache._where = L.KVCacheDesc(), 64
    return cache


def test_a_cache_of_another_device_is_refused():
    on = lambda device: SimpleNamespace(get_device=lambda: device)  # noqa: E731
    cache = bare_cache(1)
    assert cache._address(on(1)) == 64 and cache._use(1, False) is cache._desc
    for call in (lambda: cache._address(on(0)), lambda: cache._use(0, False), lambda: cache._use(0, True)):
        with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
            call()
    where = lambda *ids: [SimpleNamespace(device=torch.device("cuda", i)) for i in ids]  # noqa: E731
    serving._one_device(*where(0, 0), None, None)
    with pytest.raises(ValueError, match="more than one device: cuda:0, cuda:1"):
        serving._one_device(*where(0, 0, 1, 0))


@pytest.mark.parametrize("tokens", [1, 40])  # few rows a key head store elements, more of them vectors
def test_attention_refuses_an_output_that_vectors_cannot_reach(tokens):
    some = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(some) + 15) // 16 * 16
    d = L.TreeAttentionDesc()
    d.cache = L.KVCacheDesc(at, at, at, at, 4, 16, 2, 64, L.KV_FORMATS["int8"])
    d.batch, d.tokens, d.q_heads, d.dtype, d.scale, d.table_width = 1, tokens, 4, L.BF16, 1.0, 1
    d.q = d.page_table = d.context_lens = at
    for off in (2, 4, 8):
        d.out = at + off
        assert L.lib().ojx_tree_attention(ctypes.byref(d), None) == L.OJX_ERR_INVALID
        assert "aligned" in L.last_error()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_index_handles_are_not_computed_with(dtype):
    """At the call, not when its result is read."""
    import torchcl
    from torchcl import api

    def handle(t):  # an upload that waits for its first use
        elem, _ = api._make_handle(tuple(t.shape), t.dtype)
        elem._torchcl_host = t
        return api._wrap(elem)

    i, x = handle(torch.ones(2, 2, dtype=dtype)), handle(torch.ones(2, 2))
    calls = [lambda: torchcl.add(i, i), lambda: torchcl.mul(x, i), lambda: torchcl.sub(i, x), lambda: torchcl.relu(i), lambda: torchcl.transpose(i),
             lambda: torchcl.matmul(i, i), lambda: i + i, lambda: torchcl.add(torchcl.matmul(x, x), i), lambda: -i]
    for call in calls:
        with pytest.raises(ValueError, match="unsupported dtype"):
            call()
    torchcl.transpose(x)
    for other in (torch.float64, torch.uint8, torch.bool, torch.int16):
        with pytest.raises(ValueError, match="unsupported dtype"):
            torchcl.to_opencl(torch.ones(2, dtype=other))
