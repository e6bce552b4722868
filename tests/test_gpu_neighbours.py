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
