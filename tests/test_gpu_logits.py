"""Biases, repetition penalties and grammar masks on logits against the 64-bit formula (tests/kv_ref.py).

A column's value goes through at most five fp32 roundings (bias, quotient, count times frequency, plus presence, difference),
each half a step relative to a partial result: the bar is 5 * 2^-24 times the sum of the magnitudes."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def run(rmi, x, hist=(), hist_len=None, window=0, draft=(), masks=(), rep=1.0, pres=0.0, freq=0.0, ids=(), vals=(), allow=None, pad=0,
        in_place=False, offset=0):
    ncols, n = x.shape
    stride = n + pad
    buf = np.full((ncols, stride), 3.5, np.float32)
    buf[:, :n] = x
    flat = torch().full((ncols * stride + offset,), 3.5, device="cuda:0")
    src = flat[offset:]
    src.copy_(torch().from_numpy(buf.reshape(-1)))
    out = src if in_place else torch().full((ncols * stride + offset,), 3.5, device="cuda:0")[offset:]
    hist, draft = np.array(hist, np.int32), np.array(draft, np.int32)
    rmi.logits_process(src, n, ncols, stride, out, stride, dev(hist) if len(hist) else None,
                       dev(np.array([len(hist) if hist_len is None else hist_len], np.int32)) if len(hist) else None, len(hist), window,
                       dev(draft) if len(draft) else None, dev(np.array(masks, np.uint64).view(np.int64)) if len(draft) else None, len(draft),
                       rep, pres, freq, dev(np.array(ids, np.int32)) if len(ids) else None, dev(np.array(vals, np.float32)) if len(ids) else None,
                       len(ids), dev(allow.view(np.int32)) if allow is not None else None, allow.shape[1] if allow is not None else 0)
    got = host(out).reshape(ncols, stride)
    assert (got[:, n:] == 3.5).all()
    return got[:, :n]


def check(rmi, x, **kw):
    got = run(rmi, x, **kw)
    f32 = lambda v: np.float64(np.float32(v))  # noqa: E731
    hist = list(kw.get("hist", ()))
    used = kw.get("hist_len")
    hist = hist[:max(0, min(used, len(hist)))] if used is not None else hist
    draft = list(kw.get("draft", ()))
    masks = list(kw.get("masks", ())) or [0] * len(x)
    rep, pres, freq = (f32(kw.get(k, d)) for k, d in (("rep", 1.0), ("pres", 0.0), ("freq", 0.0)))
    vals = [f32(v) for v in kw.get("vals", ())]
    want = ref.logits(x, hist, kw.get("window", 0), draft, masks, rep, pres, freq, kw.get("ids", ()), vals, kw.get("allow"))
    big = np.abs(x.astype(np.float64)) + (max(map(abs, vals)) if vals else 0)
    bar = 5 * 2.0 ** -24 * (big * max(rep, 1 / rep) + abs(pres) + abs(freq) * (len(hist) + len(draft)))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    assert (np.abs(got[~inf] - want[~inf]) <= bar[~inf]).all()
    return got


@pytest.mark.parametrize("n", [1, 31, 1000, 1024, 1025, 5003, 248320])
def test_all_of_it(rmi, n):
    rng = np.random.default_rng(n)
    ncols = 3 if n > 10000 else 7
    x = (3 * rng.standard_normal((ncols, n))).astype(np.float32)
    hist = np.minimum(rng.zipf(1.3, 777), n) - 1
    draft = np.minimum(rng.zipf(1.3, ncols), n) - 1
    ids = rng.integers(0, n, 50)   # the same id twice: the last counts
    allow = rng.integers(0, 2 ** 32, (ncols, (n + 31) // 32), dtype=np.uint64).astype(np.uint32)
    kw = dict(hist=hist, draft=draft, masks=ref.tree_masks(rng, ncols)[0], rep=1.3, pres=0.5, freq=0.25, ids=ids, vals=rng.standard_normal(50),
              allow=allow)
    for extra in ({}, {"window": 100}, {"pad": 1}, {"pad": 4, "in_place": True}, {"offset": 1}):
        check(rmi, x, **{**kw, **extra})


@pytest.mark.parametrize("window", [1, 2, 3, 5, 8, 30, 64, 1000])
@pytest.mark.parametrize("hist", [0, 1, 4, 29, 70])
def test_windows_over_history_and_path(rmi, window, hist):
    """few tokens, so that every count changes with the window; paths longer than the window among them"""
    rng = np.random.default_rng(window * 100 + hist)
    n, ncols = 40, 12
    x = rng.standard_normal((ncols, n)).astype(np.float32)
    check(rmi, x, hist=rng.integers(0, 9, hist), window=window, draft=rng.integers(0, 9, ncols), masks=ref.tree_masks(rng, ncols, 3)[0],
          rep=2.0, pres=0.25, freq=0.5)


def test_64_columns_of_a_chain(rmi):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((64, 2050)).astype(np.float32)
    for window in (0, 20):
        check(rmi, x, hist=rng.integers(0, 2050, 500), draft=rng.integers(0, 50, 64), masks=[(2 << i) - 1 for i in range(64)], rep=1.1,
              pres=0.125, freq=0.0625, window=window)


def test_a_tree_nodes_column_is_the_column_behind_its_path(rmi):
    """the logits at a node equal, bit for bit, those of a plain call whose history ends with the node's path"""
    rng = np.random.default_rng(3)
    n, k = 3000, 9
    x = rng.standard_normal((k, n)).astype(np.float32)
    hist, draft = rng.integers(0, 60, 200), rng.integers(0, 60, k)
    masks, _ = ref.tree_masks(rng, k)
    for window in (0, 16):
        kw = dict(rep=1.2, pres=0.3, freq=0.7, window=window)
        tree = run(rmi, x, hist=hist, draft=draft, masks=masks, **kw)
        for c in range(k):
            path = [draft[j] for j in range(k) if masks[c] >> j & 1]
            one = run(rmi, x[c:c + 1], hist=np.concatenate([hist, path]), **kw)
            assert np.array_equal(one[0].view(np.uint32), tree[c].view(np.uint32))


def test_nothing_to_do_and_odd_inputs(rmi):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 100)).astype(np.float32)
    assert np.array_equal(run(rmi, x), x)
    # ids outside the vocabulary count for nothing, a history's length is clamped to its buffer and to zero
    bad = [-1, 100, 2 ** 31 - 1, -2 ** 31, 5]
    check(rmi, x, hist=bad, pres=1.0, ids=[-7, 100, 2 ** 31 - 1, 6], vals=[1.0, 2.0, 3.0, 4.0], draft=bad, masks=[31, 0])
    for used in (-5, 0, 3, 99):
        check(rmi, x, hist=[1, 2, 3, 4], hist_len=used, pres=1.0, freq=0.5)


def test_values_that_are_not_finite(rmi):
    x = np.array([[np.inf, -np.inf, np.nan, 1.0, -1.0, np.inf]], np.float32)
    got = run(rmi, x, hist=[0, 1, 2, 3, 4], rep=2.0, pres=0.5, freq=0.25, allow=np.array([[0b011111]], np.uint32))
    assert got[0, 0] == np.inf and got[0, 1] == -np.inf and np.isnan(got[0, 2])
    assert got[0, 3] == np.float32(-0.25) and got[0, 4] == np.float32(-2.75) and got[0, 5] == -np.inf


def test_a_grammar_that_allows_nothing(rmi):
    """every logit is -infinity, and argmax still answers with a token (the lowest)"""
    n = 5000
    x = empty(2 * n)
    x.normal_()
    allow = np.zeros((2, (n + 31) // 32), np.uint32)
    allow[1, 100] = 1 << 7
    rmi.logits_process(x, n, 2, n, x, n, None, None, 0, allow=dev(allow.view(np.int32)), allow_stride=allow.shape[1])
    assert np.isneginf(host(x)[:n]).all()
    idx, ws = empty(2, "int32"), empty(rmi.argmax_workspace_bytes(2), "uint8")
    rmi.argmax(x, n, idx, ws, 2, n)
    assert host(idx)[1] == 3207


def test_graph_replays_follow_the_history(rmi):
    t = torch()
    rng = np.random.default_rng(7)
    n = 4100
    x = rng.standard_normal((2, n)).astype(np.float32)
    hist = rng.integers(0, n, 64).astype(np.int32)
    dx, dh, dl, out = dev(x), dev(hist), dev(np.array([0], np.int32)), empty(2 * n)

    def step():
        rmi.logits_process(dx, n, 2, n, out, n, dh, dl, 64, repetition=1.5, presence=0.5, frequency=0.25)

    step()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=t.cuda.Stream()):
        step()
    for used in (0, 5, 64, 1):
        dl.fill_(used)
        out.zero_()
        g.replay()
        want = run(rmi, x, hist=hist, hist_len=used, rep=1.5, pres=0.5, freq=0.25)
        assert np.array_equal(host(out).reshape(2, n), want)
