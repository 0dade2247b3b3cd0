"""What the serving operators refuse and how they fail: failures inside a gradient."""
import subprocess
import sys
import textwrap

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


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
                 "ojx_kv_read", "ojx_tree_attention", "ojx_verify_drafts", "ojx_last_error")
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
