"""Outputs next to, between and (where a call allows it) on its inputs."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, host

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
