"""The example that trains with qk_norm_rope and generates from draft trees."""
import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "speculative_decode.py"
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("format,slack", [("float16", 0.05), ("int8", 0.25)])
def test_greedy_generation_follows_the_model(example, format, slack):
    """Each generated token is the likeliest one of a plain pass over the sequence, up to
    what rounding can do to its logit: q, k and v are rounded to 2^-11 (f16) of their size
    and, int8, k and v to 2^-8 of their row's largest; logits are a few units large and see
    two such layers, so 0.05 and 0.25 leave a factor of about eight."""
    r = example.main(format)
    assert r["losses"][-1] < 0.5 * r["losses"][0]
    assert r["passes"] < r["plain_passes"] == 64
    for tokens in (r["tokens"], r["plain"]):
        whole = torch.cat([r["prompts"], torch.tensor(tokens, device="cuda")], dim=1)
        with torch.no_grad():
            logits = r["model"](whole[:, :-1])[:, r["prompts"].shape[1] - 1:]
        chosen = logits.gather(2, torch.tensor(tokens, device="cuda")[:, :, None])[:, :, 0]
        assert bool((chosen >= logits.amax(2) - slack).all())


def test_sampled_generation(example):
    r = example.main("float8", temperature=0.7, new_tokens=24, batch=3)
    assert all(len(t) == 24 for t in r["tokens"]) and r["passes"] <= r["plain_passes"] == 24
    assert all(0 <= i < example.VOCAB for t in r["tokens"] for i in t)
