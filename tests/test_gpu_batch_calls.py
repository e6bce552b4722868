"""Batch attention called as its header allows and seldom is: one output of the two, rows apart, a first row of later requests, splits far
past the context, as many prompts as there may be."""
import numpy as np
import pytest

from . import batch_exact as exact
from . import batch_ref as ref
from . import kv_ref
from .gpu_util import torch
from .test_gpu_batch_attn import TYPES, Batch, ints

pytestmark = pytest.mark.gpu
F16, I8, I4 = kv_ref.F16, kv_ref.I8, kv_ref.I4


@pytest.fixture(scope="module")
def rmi():
    torch()
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


LENS = [(300, 1), (700, 6), (1100, 40), (0, 9)]


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("split", [128, 384, 1152])
@pytest.mark.parametrize("lens", [LENS, LENS[:2]])
def test_one_output_and_rows_apart(rmi, kt, vt, split, lens):
    """y alone, Q8_1 alone, both with rows apart: the bytes of both together; nothing between the rows"""
    t = torch()
    b = Batch(np.random.default_rng(split), lens, kt, vt, 2, 4, 128, 32)
    b.run(rmi, split)
    y, blocks, n = b.y.clone(), b.blocks.clone(), int(b.start[-1])
    width, raw = b.nh * b.hd, b.blocks.shape[1]
    for pad_y, pad_q in ((0, None), (None, 0), (12, 8), (12, None), (None, 8)):
        args = list(b.args)
        got = None if pad_y is None else t.full((b.ntok, width + pad_y), 77.0, dtype=y.dtype, device="cuda")
        got8 = None if pad_q is None else t.full((b.ntok, raw + pad_q), 0xee, dtype=t.uint8, device="cuda")
        args[11:15] = [got, width + (pad_y or 0), got8, raw + (pad_q or 0)]
        rmi.gqa_paged_attn(*args)
        t.cuda.synchronize()
        if got is not None:
            assert t.equal(got[:, :width], y.view(b.ntok, width)) and bool((got[:, width:] == 77.0).all()) and bool((got[n:] == 77.0).all())
        if got8 is not None:
            assert t.equal(got8[:, :raw], blocks) and bool((got8[:, raw:] == 0xee).all())


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4)])
@pytest.mark.parametrize("split", [128, 2048])
def test_a_part_of_a_batch(rmi, kt, vt, split):
    """calls on the first and the other requests of a batch, over the same rows: those of the other part stay as they are"""
    t = torch()
    lens = [(1300, 2), (40, 33), (1200, 1), (600, 5), (9, 0), (80, 70)]
    b = Batch(np.random.default_rng(7), lens, kt, vt, 2, 4, 128, 64)
    whole, _ = b.run(rmi, split)
    for cut in (1, 3, 5):
        y = t.full_like(b.y, 77.0)
        for part in (slice(cut, None), slice(0, cut)):
            args = list(b.args)
            args[5] = b.args[5][part].contiguous()
            args[7] = ints(b.start[part.start:part.stop + 1 if part.stop else None])
            args[8] = b.args[8][part].contiguous()
            args[11], args[13], args[16] = y, None, len(lens[part])
            rmi.gqa_paged_attn(*args)
            t.cuda.synchronize()
            if part.start:   # so far the rows of the requests from `cut` on
                first = int(b.start[cut])
                assert bool((y[:first] == 77.0).all()) and np.array_equal(y[first:].double().cpu().numpy(), whole[first:])
        assert np.array_equal(y.double().cpu().numpy(), whole)


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I8)])
def test_splits_past_the_context(rmi, kt, vt):
    for lens in (LENS, LENS[:1]):
        b = Batch(np.random.default_rng(3), lens, kt, vt, 2, 4, 128, 32)
        first, blocks = b.run(rmi, 1280)
        b.check(first, blocks)
        for split in (1 << 30, (1 << 31) - 128):
            assert rmi.gqa_paged_workspace_bytes(b.ntok, 1140, b.nh, b.hd, split) == 16
            y, again = b.run(rmi, split)
            assert np.array_equal(y, first) and np.array_equal(again, blocks)


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("most", [3, 200])
def test_most_prompts(rmi, name, most):
    """4096 prompts of up to three rows, one of 200 among them (left out where the bound says so)"""
    t = torch()
    rng = np.random.default_rng(most)
    lens = rng.integers(0, 4, 4096)
    lens[2777] = 200
    start = np.concatenate([[5], 5 + np.cumsum(lens)])   # five rows before the first
    n, hd, G = int(start[-1]) + 4, 128, 4
    q, k, v = (t.from_numpy(rng.standard_normal((n, h, hd)).astype(np.float32)).to(getattr(t, name)).cuda() for h in (G, 1, 1))
    y = t.full_like(q, 77.0)
    scale = float(np.float32(hd ** -0.5))
    rmi.gqa_prompt_attn(q, G * hd, k, hd, v, hd, ints(start), None, 0, y, G * hd, None, 0, 4096, n, most, G, 1, hd, scale)
    got = y.double()
    assert bool((got[:5] == 77.0).all()) and bool((got[start[-1]:] == 77.0).all())
    if most < 200:
        assert bool((got[start[2777]:start[2778]] == 77.0).all())
    for i in [0, 1, 63, 64, 65, 1000, 2776, 2777, 2778, 4094, 4095] + rng.integers(0, 4096, 60).tolist():
        if 0 < lens[i] <= most:
            r = slice(int(start[i]), int(start[i + 1]))
            want, bound = exact.attention(q[r].double(), k[r].double(), v[r].double(), t.arange(int(lens[i]), device="cuda"), scale, ref.HALF_STEP[name],
                                          ref.HALF_STEP[name])
            assert exact.outside(got[r], want, bound) == 0
    done = np.concatenate([np.arange(start[i], start[i + 1]) for i in range(4096) if lens[i] <= most])
    assert bool((got[t.from_numpy(done).cuda()] != 77.0).any(-1).all())
