"""Outputs next to, between and (where a call allows it) on its inputs."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host
from tests.test_gpu_tree_attn import Call, as_masks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


@pytest.mark.parametrize("first", [17, 35])
def test_rows_copied_within_an_fp16_cache(rmi, first):
    """source and destination side by side in one cache"""
    max_ctx, nkv, hd, n = 50, 2, 128, 9
    x = np.random.default_rng(1).standard_normal((max_ctx, nkv, hd)).astype(np.float16)
    cache = dev(x.view(np.uint16))
    rmi.kv_write(ref.F16, cache[26:26 + n], nkv * hd, cache, first, n, nkv, hd, max_ctx)
    x[first:first + n] = x[26:26 + n].copy()
    assert np.array_equal(host(cache).view(np.float16), x)
    out = cache[:n]
    rmi.kv_read(ref.F16, cache, out, nkv * hd, 9, n, nkv, hd, max_ctx)
    x[:n] = x[9:9 + n].copy()
    assert np.array_equal(host(cache).view(np.float16), x)


def test_logits_between_the_columns(rmi):
    """outputs in the gaps of the columns' stride"""
    rng, n, ncols = np.random.default_rng(2), 1003, 5
    x = rng.standard_normal((ncols, n)).astype(np.float32)
    buf = np.zeros((ncols, 2 * n), np.float32)
    buf[:, :n] = x
    d = dev(buf.reshape(-1))
    hist = rng.integers(0, n, 700)
    rmi.logits_process(d, n, ncols, 2 * n, d[n:], 2 * n, dev(hist.astype(np.int32)), dev(np.array([700], np.int32)), 700, presence=0.5)
    got = host(d).reshape(ncols, 2 * n)
    want = np.where(np.bincount(hist, minlength=n) > 0, x - np.float32(0.5), x)
    assert np.array_equal(got[:, :n], x) and np.array_equal(got[:, n:], want)


@pytest.mark.parametrize("types", [(ref.F16, ref.F16), (ref.I8, ref.I4)], ids=["f16", "i8_i4"])
@pytest.mark.parametrize("nh,nkv,hd,ntok,base,nsub", [(16, 4, 256, 1, 300, 1), (4, 2, 128, 3, 20, 1), (4, 2, 256, 6, 1300, 1), (4, 2, 256, 6, 20, 1),
                                                      (8, 2, 256, 6, 20, 7), (8, 2, 128, 6, 1000, 6), (4, 2, 256, 20, 20, 1), (4, 2, 128, 30, 90, 1),
                                                      (4, 2, 256, 40, 20, 1), (4, 1, 256, 33, 400, 1)])
def test_tree_results_in_the_queries_place(rmi, types, nh, nkv, hd, ntok, base, nsub):
    """y is q: every form, one chunk and several, rows that do not fill a group"""
    masks, _ = ref.tree_masks(np.random.default_rng(ntok), ntok)
    for m in (masks, None):
        c = Call(rmi, types, nh, nkv, hd, ntok, base, m, nsub=nsub)
        want = c.run()
        q = dev(c.q)
        ws = empty(rmi.gqa_tree_workspace_bytes(c.max_ctx, nh, nkv, hd, ntok, nsub), "uint8")
        rmi.gqa_tree_decode(q, types[0], dev(c.raw[0]), types[1], dev(c.raw[1]), dev(np.array([base], np.int32)), as_masks(m), dev(c.q3), c.width, q,
                            nh * hd, None, 0, ws, nh, nkv, hd, ntok, c.max_ctx, nsub, c.scale)
        assert np.array_equal(host(q).reshape(want.shape).view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("nh,ntok", [(2, 1), (2, 7), (3, 5)])
def test_q8_rows_between_the_gates(rmi, orc, nh, ntok):
    """rows of Q8_1 in the place of a head's spent q, between the gates of two heads"""
    hd, base = 256, 130
    c = Call(rmi, (ref.I8, ref.I8), nh, nh, hd, ntok, base, None, nsub=1)
    want = np.stack([orc.quantize_q8_1(y.reshape(-1), nh * hd) for y in c.run()])
    d = dev(c.q3.reshape(-1))
    ws = empty(rmi.gqa_tree_workspace_bytes(c.max_ctx, nh, nh, hd, ntok, 1), "uint8")
    rmi.gqa_tree_decode(dev(c.q), ref.I8, dev(c.raw[0]), ref.I8, dev(c.raw[1]), dev(np.array([base], np.int32)), None, d, c.width, None, 0, d[2 * hd:],
                        4 * c.width, ws, nh, nh, hd, ntok, c.max_ctx, 1, c.scale)
    got = host(d).reshape(ntok, c.width)
    n = nh * hd // 32 * 9   # words of a row
    assert np.array_equal(got[:, 2 * hd:2 * hd + n].copy().view(np.uint8).reshape(ntok, -1), want)
    got[:, 2 * hd:2 * hd + n] = c.q3[:, 2 * hd:2 * hd + n]
    assert np.array_equal(got, c.q3)
    with pytest.raises(ValueError, match="gates"):
        rmi.gqa_tree_decode(dev(c.q), ref.I8, dev(c.raw[0]), ref.I8, dev(c.raw[1]), dev(np.array([base], np.int32)), None, d, c.width, None, 0,
                            d[3 * hd - 1:], 4 * c.width, ws, nh, nh, hd, ntok, c.max_ctx, 1, c.scale)


def test_tree_results_beside_the_gates(rmi):
    """y in the columns behind a buffer's gates"""
    nh, nkv, hd, ntok, base = 4, 2, 256, 9, 130
    c = Call(rmi, (ref.I8, ref.I8), nh, nkv, hd, ntok, base, None, nsub=1)
    want = c.run()
    width = 2 * nh * hd + nh * hd
    buf = np.zeros((ntok, width), np.float32)
    buf[:, :2 * nh * hd] = c.q3[:, :2 * nh * hd]
    d = dev(buf.reshape(-1))
    ws = empty(rmi.gqa_tree_workspace_bytes(c.max_ctx, nh, nkv, hd, ntok, 1), "uint8")
    rmi.gqa_tree_decode(dev(c.q), ref.I8, dev(c.raw[0]), ref.I8, dev(c.raw[1]), dev(np.array([base], np.int32)), None, d, width, d[2 * nh * hd:], width,
                        None, 0, ws, nh, nkv, hd, ntok, c.max_ctx, 1, c.scale)
    got = host(d).reshape(ntok, width)
    assert np.array_equal(got[:, 2 * nh * hd:].reshape(want.shape).view(np.uint32), want.view(np.uint32))
    assert np.array_equal(got[:, :2 * nh * hd], buf[:, :2 * nh * hd])
