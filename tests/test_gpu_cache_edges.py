"""The cache operators where their kernels change course: lists of several blocks, budgets at a block's end."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_cache as T  # noqa: E402
from test_gpu_cache import BF16, F16  # noqa: E402

GUARD = 1 << 18  # bytes on either side of a workspace


@pytest.fixture
def guarded(monkeypatch):
    """Workspaces between guard bytes, which are as they were when the test ends."""
    made = []

    def buffer(n):
        whole = torch.full((max(n, 16) + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
        made.append((whole, max(n, 16)))
        return whole[GUARD:GUARD + max(n, 16)]

    monkeypatch.setattr(T, "buffer", buffer)
    yield
    torch.cuda.synchronize()
    assert made
    for whole, n in made:
        assert torch.all(whole[:GUARD] == 0xA5) and torch.all(whole[GUARD + n:] == 0xA5), "a byte outside a workspace changed"


def few_values(w, rng):
    w[:] = rng.integers(0, 700, w.shape)


LONG = [
    dict(ctx=[40000], budget=32767),
    dict(ctx=[40000], budget=32768),
    dict(ctx=[40000, 36000], budget=32769, recent=300, sinks=4, moved=True),
    dict(ctx=[33000, 40000], budget=33000, recent=100),
    dict(ctx=[40000], budget=33000, weigh=few_values),
    dict(ctx=[70001], budget=40000, sinks=2),
    dict(ctx=[70001, 9], budget=65536, moved=True),
    dict(ctx=[100000], budget=70000, recent=1000, max_ctx=98000),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: f"n{max(c['ctx'])}to{c['budget']}")
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_lists_of_several_blocks(guarded, case, in_place):
    """Distinct weights, so that the selection ends without a tie, and the budget past the first block's rows."""
    T.run_evict(dt=F16 if in_place else BF16, dim=64, kv=2, seed=70, in_place=in_place,
                **dict(dict(weigh=lambda w, rng: w.__setitem__(..., rng.permutation(w.size).reshape(w.shape))), **case))
