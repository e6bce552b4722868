"""The bound of tests/batch_exact.py sees what a kernel might lose (mistakes planted in the formula, on the CPU)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from . import batch_exact as exact  # noqa: E402


def rows(seed, n, heads, n_kv, dims, at):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(len(at), heads, dims, generator=g, dtype=torch.float64)
    k, v = (torch.randn(n, n_kv, dims, generator=g, dtype=torch.float64) for _ in range(2))
    gate = torch.randn(len(at), heads, dims, generator=g, dtype=torch.float64)
    return q, k, v, gate, torch.tensor(at)


@pytest.mark.parametrize("n,step,lost", [(9001, 2.0 ** -11, 128), (9001, 2.0 ** -11, 32), (1101, 2.0 ** -11, 1), (1101, 2.0 ** -8, 32), (8001, 2.0 ** -8, 128)])
def test_a_lost_part_is_outside(n, step, lost):
    q, k, v, gate, at = rows(n + lost, n, 4, 1, 128, [n - 1])
    args = q, k, v, at, 128 ** -0.5, step, step
    want, bound = exact.attention(*args, gate=gate, depth=n / 4)
    part = torch.arange(n // 3, n // 3 + lost)
    wrong, _ = exact.attention(*args, gate=gate, left_out=part)
    assert exact.outside(wrong, want, bound) > 0
    if lost > 1:
        assert exact.outside(wrong, want, bound) > 10


@pytest.mark.parametrize("n,dims,by", [(700, 128, 1), (4090, 128, 32), (1000, 256, 3), (1, 128, 1)])
def test_marks(n, dims, by):
    pos = torch.arange(n)
    assert torch.equal(exact.marked(pos, dims, by).double(), exact.marks(n, dims, by).cumsum(0))


def test_agrees_with_the_plain_restatement():
    from . import batch_ref as ref
    q, k, v, gate, at = rows(3, 150, 6, 2, 128, [140, 141, 149])
    want, bound = exact.attention(q[:2], k, v, at[:2], 128 ** -0.5, 2.0 ** -11, 2.0 ** -11, gate=gate[:2])
    plain, wide = ref.attention(q[:2].numpy(), k.numpy(), v.numpy(), 140, 128 ** -0.5, gate[:2].numpy(), 2.0 ** -11, 2.0 ** -11)
    assert np.abs(want.numpy() - plain).max() < 1e-14 and (bound.numpy() < wide).all()
