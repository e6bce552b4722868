"""Calls of rmi_logits_process at the edges of what its arguments may be."""
import numpy as np
import pytest

from tests.gpu_util import dev, empty, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def test_no_history(rmi):
    """without a capacity there is no history, whatever the pointers: null or not; with one, both are needed"""
    n, rng = 1500, np.random.default_rng(1)
    x = rng.standard_normal((2, n)).astype(np.float32)
    d, out = dev(x), empty(2 * n)
    for hist, length in ((None, None), (dev(np.arange(9, dtype=np.int32)), dev(np.array([9], np.int32))), (dev(np.arange(9, dtype=np.int32)), None)):
        out.zero_()
        rmi.logits_process(d, n, 2, n, out, n, hist, length, 0, presence=1.0, frequency=2.0, repetition=3.0)
        assert np.array_equal(host(out).reshape(2, n), x)
    for hist, length in ((None, None), (None, dev(np.array([9], np.int32))), (dev(np.arange(9, dtype=np.int32)), None)):
        with pytest.raises(ValueError, match="null"):
            rmi.logits_process(d, n, 2, n, out, n, hist, length, 9)


def test_ids_outside_the_vocabulary_fill_the_window(rmi):
    n = 40
    x = np.zeros((1, n), np.float32)
    hist = np.array([3, 4, -1, 99, 5], np.int32)
    out = empty(n)
    for window, hit in ((0, [3, 4, 5]), (1, [5]), (3, [5]), (4, [4, 5])):
        rmi.logits_process(dev(x), n, 1, n, out, n, dev(hist), dev(np.array([5], np.int32)), 5, window, presence=1.0)
        assert sorted(np.nonzero(host(out))[0]) == hit


@pytest.mark.parametrize("n", [7, 5000, 70001])
def test_argmax_of_columns_that_a_grammar_empties(rmi, n):
    """every logit -infinity: the lowest token; one token allowed: that one, whatever its logit"""
    words = (n + 31) // 32
    allow = np.zeros((3, words), np.uint32)
    one = n - 2
    allow[1, one // 32] = np.uint32(1 << one % 32)
    allow[2] = 0xffffffff
    x = np.random.default_rng(n).standard_normal((3, n)).astype(np.float32)
    x[1, one] = -1e30
    out, idx, ws = empty(3 * n), empty(3, "int32"), empty(rmi.argmax_workspace_bytes(3), "uint8")
    rmi.logits_process(dev(x), n, 3, n, out, n, None, None, 0, allow=dev(allow.view(np.int32)), allow_stride=words)
    z = host(out).reshape(3, n)
    assert np.isneginf(z[0]).all() and np.isneginf(np.delete(z[1], one)).all() and z[1, one] == np.float32(-1e30)
    assert np.array_equal(z[2], x[2])
    idx.fill_(-7)
    rmi.argmax(out, n, idx, ws, 3, n)
    assert list(host(idx)) == [0, one, int(x[2].argmax())]
