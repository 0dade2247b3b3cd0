"""The serving operators beside other work: caches made on torchcl's stream and used on
torch's."""
import pytest
import torch

from test_gpu_serving import pages_for, rnd

pytestmark = pytest.mark.gpu
LONG = 200_000_000  # clocks of a wait on a stream: about a tenth of a second


@pytest.fixture(scope="module")
def S():
    from torchcl import serving
    return serving


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
