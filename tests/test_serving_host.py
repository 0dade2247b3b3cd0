"""The serving operators without a GPU: refusals before any device work, masks and tables,
and the plain verification reference's own distribution."""
import ctypes

import numpy as np
import pytest
import torch

import serving_reference as ref
from torchcl import _lib as L
from torchcl import serving


def test_tree_mask():
    m = serving.tree_mask([-1, 0, 0, 1, -1])
    assert m.shape == (5, 1) and m[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000]
    batch = serving.tree_mask(torch.tensor([[-1, 0, 1], [-1, 0, 0]]))
    assert batch[:, :, 0].tolist() == [[1, 3, 7], [1, 3, 5]]
    chain = serving.tree_mask([i - 1 for i in range(130)])
    assert chain.shape == (130, 3)
    assert torch.equal(ref.words_to_bool(chain, 130), torch.ones(130, 130).tril().bool())
    for bad in ([0], [-1, 1], [-1, 0, 5]):
        with pytest.raises(ValueError):
            serving.tree_mask(bad)
    assert serving.tree_mask(torch.zeros(2, 0, dtype=torch.int32)).shape == (2, 0, 0)


def test_rope_table():
    t = serving.rope_table(3000, 8, 100.0)
    angle = 2999 * 100.0 ** (-np.arange(0, 8, 2) / 8)
    np.testing.assert_allclose(t[2999].numpy(), np.concatenate([np.cos(angle), np.sin(angle)]), rtol=0, atol=6e-8)
    assert serving.rope_table(4, 0).shape == (4, 0)
    with pytest.raises(ValueError):
        serving.rope_table(4, 3)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="device tensor"):
        serving.qk_norm_rope(x, x, None, None, serving.rope_table(4, 64), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="device tensor"):
        serving.verify_drafts(torch.zeros(1, 1, 4), torch.zeros(1, 1), torch.zeros(1, 1), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="format"):
        serving.KVCache(4, 16, 2, 64, "int3")
    with pytest.raises(ValueError, match="multiple of 16"):
        serving.KVCache(4, 16, 2, 72)
    with pytest.raises(ValueError, match="at least one"):
        serving.KVCache(0, 16, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        serving.KVCache.from_pages(torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4, 64))


def _rejects(fn, *args):
    assert fn(*args) == L.OJX_ERR_INVALID
    return L.last_error()


def test_c_entries_refuse_bad_arguments_before_the_device():
    lib, P = L.lib(), ctypes.byref
    some = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(some) + 15) // 16 * 16
    good = L.KVCacheDesc(at, at, at, at, 4, 16, 2, 64, L.KV_FORMATS["int8"])

    def cache(**kw):
        c = L.KVCacheDesc.from_buffer_copy(good)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    rows = L.Rows(at, 128, 64)
    for bad, word in (({"format": 0}, "format"), ({"format": 9}, "format"), ({"head_dim": 24}, "head_dim"), ({"head_dim": 528}, "head_dim"),
                      ({"page_size": 0}, "at least one"), ({"k": at + 2}, "aligned"), ({"v": None}, "aligned"), ({"k_scale": None}, "steps"),
                      ({"num_pages": 1 << 40}, "pages")):
        assert word in _rejects(lib.ojx_kv_append, P(cache(**bad)), P(rows), P(rows), L.F32, 1, at, 0, None)
    assert "NULL" in _rejects(lib.ojx_kv_append, None, P(rows), P(rows), L.F32, 1, at, 0, None)
    assert "dtype" in _rejects(lib.ojx_kv_append, P(good), P(rows), P(rows), 5, 1, at, 0, None)
    assert "negative" in _rejects(lib.ojx_kv_append, P(good), P(rows), P(rows), L.F32, -1, at, 0, None)
    assert "NULL" in _rejects(lib.ojx_kv_append, P(good), P(rows), None, L.F32, 1, at, 0, None)
    assert "aligned" in _rejects(lib.ojx_kv_read, P(good), at + 4, at, L.F32, 1, at, 0, None)
    assert "NULL" in _rejects(lib.ojx_kv_keep_path, P(good), at, 1, at, at, None, 1, 1, None)
    assert lib.ojx_kv_append(P(good), P(rows), P(rows), L.F32, 0, None, 0, None) == L.OJX_OK

    q = L.QkDesc()
    q.tokens, q.q_heads, q.kv_heads, q.head_dim, q.rotary_dim = 1, 1, 1, 64, 64
    for name, value, word in (("head_dim", 63, "head_dim"), ("head_dim", 514, "head_dim"), ("rotary_dim", 66, "rotary_dim"),
                              ("rotary_dim", 3, "rotary_dim"), ("dtype", 7, "dtype"), ("tokens", -1, "negative"), ("eps", -1.0, "eps"),
                              ("eps", float("nan"), "eps"), ("dtype", L.BF16, "NULL")):
        d = L.QkDesc.from_buffer_copy(q)
        setattr(d, name, value)
        assert word in _rejects(lib.ojx_qk_norm_rope, P(d), at, at, None)
        assert word in _rejects(lib.ojx_qk_norm_rope_backward, P(d), None, None, at, at, None, None, None)
    q.q = q.k = rows
    q.positions = q.table = at
    assert "holds" in _rejects(lib.ojx_qkv_to_cache, P(q), P(rows), at, P(cache(head_dim=128)), at, 0, None)

    t = L.TreeAttentionDesc()
    t.cache, t.batch, t.tokens, t.q_heads, t.dtype, t.scale, t.table_width = good, 1, 1, 4, L.BF16, 1.0, 1
    for name, value, word in (("cache", cache(head_dim=96), "64 or 128"), ("dtype", L.F32, "bf16 or fp16"), ("q_heads", 3, "evenly"),
                              ("cache", cache(format=L.F16), "dtype"), ("scale", 0.0, "scale"), ("scale", float("nan"), "scale"),
                              ("batch", -1, "negative"), ("q", None, "NULL")):
        d = L.TreeAttentionDesc.from_buffer_copy(t)
        setattr(d, name, value)
        assert word in _rejects(lib.ojx_tree_attention, P(d), None)
    t.batch = 0
    assert lib.ojx_tree_attention(P(t), None) == L.OJX_OK

    v = L.VerifyDesc()
    v.batch, v.tokens, v.vocab = 1, 1, 8
    for name, value, word in (("tokens", 0, "nodes"), ("tokens", 2000, "nodes"), ("vocab", 0, "vocabulary"), ("vocab", 1 << 30, "vocabulary"),
                              ("dtype", 4, "dtype"), ("batch", -1, "negative"), ("target", None, "NULL")):
        d = L.VerifyDesc.from_buffer_copy(v)
        setattr(d, name, value)
        assert word in _rejects(lib.ojx_verify_drafts, P(d), None)


def test_reference_verification_emits_the_target():
    """The walk's first emitted token, by integration over a grid of the random numbers,
    has the target's distribution (one sibling, three tokens)."""
    p, q = np.array([[0.5, 0.3, 0.2]] * 2, np.float32), np.array([[0.2, 0.2, 0.6]] * 2, np.float32)
    share, n = np.zeros(3), 100
    for x in range(3):
        for a in range(n):
            for b in range(n):
                path, nxt = ref.verify(p, [0, x], [-1, 0], np.array([(b + 0.5) / n, (a + 0.5) / n], np.float32), q)
                share[x if len(path) == 2 else nxt] += q[0, x] / n ** 2
    np.testing.assert_allclose(share, p[0], atol=2.5 / n)
