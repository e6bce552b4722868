"""The 16-, 8- and 4-bit K/V caches: rows written and read back, the fused norm + rotation + write, the accepted path's move.

Codes and scales are equal to the 64-bit restatement's (tests/kv_ref.py), bit for bit: the scale is decided exactly, codes
are rounded as if divided exactly, and quantised K rows are normed and rotated in fp64."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu

TYPES = [ref.F16, ref.I8, ref.I4]
GUARD = 64


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def new_cache(rmi, type_, max_ctx, n_kv, hd, fill=0x5a):
    """a cache between guard bytes: (whole buffer, cache view)"""
    n = rmi.kv_cache_bytes(type_, max_ctx, n_kv, hd)
    whole = torch().full((n + 2 * GUARD,), fill, dtype=torch().uint8, device="cuda:0")
    return whole, whole[GUARD:GUARD + n]


def changed_positions(before, after, type_, max_ctx, n_kv, hd):
    """positions with a byte that differs"""
    a, b = np.asarray(before), np.asarray(after)
    if type_ == ref.F16:
        return set(np.nonzero((a != b).reshape(max_ctx, -1).any(1))[0])
    per = hd if type_ == ref.I8 else hd // 2
    cut = n_kv * max_ctx * per
    c = (a != b)[:cut].reshape(n_kv, max_ctx, per).any((0, 2))
    s = (a != b)[cut:].reshape(n_kv, max_ctx, hd // 32).any((0, 2))
    return set(np.nonzero(c | s)[0])


def rows_in(rng, n, n_kv, hd):
    """rows of every magnitude a cache meets, with empty blocks, ties and one-sided maxima among them"""
    x = rng.standard_normal((n, n_kv, hd)).astype(np.float32)
    x *= np.exp2(rng.integers(-24, 14, (n, n_kv, hd // 32))).astype(np.float32).repeat(32, -1)
    flat = x.reshape(-1, 32)
    flat[rng.integers(0, len(flat), max(1, len(flat) // 8))] = 0
    ties = rng.integers(0, len(flat), max(1, len(flat) // 8))
    flat[ties] = rng.integers(-254, 255, (len(ties), 32)) * 0.5      # halves of a scale of 1
    flat[ties, 0] = 127.0
    one = rng.integers(0, len(flat), max(1, len(flat) // 16))
    flat[one] = 0
    flat[one, 31] = -3.25
    return x


@pytest.mark.parametrize("n_kv,hd", [(4, 256), (1, 128), (3, 128)])
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("f16", [False, True])
def test_write_and_read(rmi, type_, n_kv, hd, f16):
    rng = np.random.default_rng(11 + type_)
    max_ctx, first, n = 61, 7, 33
    x = rows_in(rng, n, n_kv, hd)
    if f16:
        x = x.astype(np.float16)
    for pad in (0, 8, 3):   # rows packed, apart and apart by an odd number of elements
        stride = n_kv * hd + pad
        src = np.zeros((n, stride), x.dtype)
        src[:, :n_kv * hd] = x.reshape(n, -1)
        whole, cache = new_cache(rmi, type_, max_ctx, n_kv, hd)
        before = host(cache).copy()
        rmi.kv_write(type_, dev(src.view(np.uint16) if f16 else src), stride, cache, first, n, n_kv, hd, max_ctx)
        after = host(cache)
        assert changed_positions(before, after, type_, max_ctx, n_kv, hd) <= set(range(first, first + n))
        assert (host(whole)[:GUARD] == 0x5a).all() and (host(whole)[-GUARD:] == 0x5a).all()
        want = ref.held(x, type_)
        got = ref.decode(after, type_, max_ctx, n_kv, hd)[first:first + n]
        assert np.array_equal(got, want)
        if type_ != ref.F16:   # the bytes themselves, not only their values
            full = np.zeros((max_ctx, n_kv, hd))
            full[first:first + n] = x
            same = ref.encode(full, type_)
            keep = changed_positions(same, after, type_, max_ctx, n_kv, hd)
            assert not keep & set(range(first, first + n))
        for out16 in (False, True):
            out = np.full((n, stride), 9, np.float16 if out16 else np.float32)
            d = dev(out.view(np.uint16) if out16 else out)
            rmi.kv_read(type_, cache, d, stride, first, n, n_kv, hd, max_ctx)
            back = host(d).view(out.dtype).reshape(n, stride)
            assert np.array_equal(back[:, :n_kv * hd].reshape(n, n_kv, hd).astype(np.float64), want)
            assert (back[:, n_kv * hd:] == 9).all()


@pytest.mark.parametrize("type_", [ref.I8, ref.I4])
def test_write_saturates_and_marks_non_finite_blocks(rmi, type_):
    x = np.zeros((5, 1, 128), np.float32)
    x[0, 0, 3] = 3e38
    x[0, 0, 4] = -3e38
    x[0, 0, 5] = 1.0
    x[1, 0, 40], x[1, 0, 41] = np.nan, 5.0
    x[2, 0, 70], x[3, 0, 127] = np.inf, -np.inf
    x[4, 0, :] = 1e-42                                              # fp32 subnormals: the smallest scale
    cache = new_cache(rmi, type_, 5, 1, 128)[1]
    rmi.kv_write(type_, dev(x), 128, cache, 0, 5, 1, 128, 5)
    raw = host(cache)
    got = ref.decode(raw, type_, 5, 1, 128)[:, 0]
    top = 127 * 512.0 if type_ == ref.I8 else 7 * 8192.0
    assert got[0, 3] == top and got[0, 4] == -top and got[0, 5] == 0
    assert np.isnan(got[1, 32:64]).all() and not got[1, :32].any() and not got[1, 64:].any()
    assert np.isnan(got[2, 64:96]).all() and np.isnan(got[3, 96:]).all()
    assert not got[4].any() and (raw[-4:] == 1).all()
    out = empty(5 * 128)
    rmi.kv_read(type_, cache, out, 128, 0, 5, 1, 128, 5)
    assert np.array_equal(host(out).reshape(5, 128).astype(np.float64), got, equal_nan=True)


@pytest.mark.parametrize("type_", TYPES)
def test_no_rows(rmi, type_):
    cache = new_cache(rmi, type_, 4, 1, 128)[1]
    before = host(cache).copy()
    x = empty(128)
    rmi.kv_write(type_, x, 128, cache, 4, 0, 1, 128, 4)
    rmi.kv_read(type_, cache, x, 128, 0, 0, 1, 128, 4)
    assert np.array_equal(before, host(cache))


# ---- norm + rotation + write ------------------------------------------------------------------------------------------

def axis_of(i, sections, interleaved):
    if interleaved:
        a = i % 3
        return a if a and i < 3 * sections[a] else 0
    return 0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2


def prep_ref(x, w, eps, n_rot, theta, sections, interleaved, axis_pos):
    """x [ntok, heads, hd] -> normed and rotated, float64"""
    x = x.astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    half = n_rot // 2
    y = x.copy()
    for i in range(half):
        p = np.asarray(axis_pos)[axis_of(i, sections, interleaved)].astype(np.float64)
        ang = p * theta ** (-2.0 * i / n_rot)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        y[..., i] = x[..., i] * c - x[..., i + half] * s
        y[..., i + half] = x[..., i] * s + x[..., i + half] * c
    return y


@pytest.mark.parametrize("ktype,vtype,nh,nkv,hd,n_rot,sections,inter,ntok,extra", [
    (ref.I8, ref.I8, 16, 4, 256, 64, (12, 10, 10), True, 1, 0),
    (ref.I8, ref.I4, 16, 4, 256, 64, (11, 11, 10), True, 5, 3),
    (ref.I4, ref.I4, 4, 2, 128, 128, (16, 24, 24), False, 67, 0),
    (ref.F16, ref.I8, 5, 1, 128, 96, (16, 16, 16), True, 9, 1),
    (ref.I8, ref.F16, 2, 2, 256, 0, (0, 0, 0), False, 3, 0),
    (ref.I8, ref.I8, 3, 3, 256, 256, (128, 0, 0), False, 130, 2),
])
def test_prep_axes(rmi, ktype, vtype, nh, nkv, hd, n_rot, sections, inter, ntok, extra):
    rng = np.random.default_rng(5)
    max_ctx, p0, theta, eps = 200, 13, 1e6, 1e-6
    width = 2 * nh * hd + 2 * nkv * hd
    q3 = rng.standard_normal((ntok, width + extra)).astype(np.float32)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32)
    axis_pos = rng.integers(-5, 70000, (3, ntok)).astype(np.int32)
    k, v = new_cache(rmi, ktype, max_ctx, nkv, hd), new_cache(rmi, vtype, max_ctx, nkv, hd)
    kb, vb = host(k[1]).copy(), host(v[1]).copy()
    qo = empty(ntok * nh * hd)
    rmi.attn_prep_axes(dev(q3), width + extra, dev(qn), dev(kn), ktype, k[1], vtype, v[1], dev(np.array([p0], np.int32)), dev(axis_pos),
                       qo, nh, nkv, hd, n_rot, theta, 1.0, 0.0, sections, inter, eps, ntok, max_ctx)
    args = (eps, n_rot, theta, sections, inter, axis_pos)
    q = q3[:, :2 * nh * hd].reshape(ntok, nh, 2, hd)[:, :, 0]
    kx, vx = (q3[:, 2 * nh * hd + i * nkv * hd:2 * nh * hd + (i + 1) * nkv * hd].reshape(ntok, nkv, hd) for i in range(2))
    # q in fp32: rsqrt (1 ulp) and the sum's 256 roundings halved by the root, two products, the rotation's two roundings
    want = prep_ref(q, qn, *args)
    assert np.abs(host(qo).reshape(want.shape) - want).max() <= (128 + 8) * 2.0 ** -24 * np.abs(want).max()
    kr = prep_ref(kx, kn, *args).astype(np.float32)
    got = ref.decode(host(k[1]), ktype, max_ctx, nkv, hd)[p0:p0 + ntok]
    assert np.array_equal(got, ref.held(kr, ktype))
    assert np.array_equal(ref.decode(host(v[1]), vtype, max_ctx, nkv, hd)[p0:p0 + ntok], ref.held(vx, vtype))
    for (whole, c), b, t in ((k, kb, ktype), (v, vb, vtype)):
        assert changed_positions(b, host(c), t, max_ctx, nkv, hd) <= set(range(p0, p0 + ntok))
        assert (host(whole)[:GUARD] == 0x5a).all() and (host(whole)[-GUARD:] == 0x5a).all()


@pytest.mark.parametrize("factor", [1.0, 4.0])
def test_prep_axes_text_positions_give_attn_preps_rows(rmi, factor):
    """q and V bit for bit; K within one fp16 step (fp64 before the rounding here, fp32 there), nearly always equal"""
    rng = np.random.default_rng(6)
    nh, nkv, hd, ntok, max_ctx, p0 = 16, 4, 256, 7, 128, 40
    width = 2 * nh * hd + 2 * nkv * hd
    q3 = dev(rng.standard_normal((ntok, width)).astype(np.float32))
    qn, kn = dev(1 + 0.1 * rng.standard_normal(hd).astype(np.float32)), dev(1 + 0.1 * rng.standard_normal(hd).astype(np.float32))
    pos = dev(np.array([p0], np.int32))
    outs = []
    for axes in (False, True):
        k, v = (torch().zeros(max_ctx * nkv * hd, dtype=torch().int16, device="cuda:0") for _ in range(2))
        qo = empty(ntok * nh * hd)
        if axes:
            rmi.attn_prep_axes(q3, width, qn, kn, ref.F16, k, ref.F16, v, pos, None, qo, nh, nkv, hd, 64, 1e7, factor, 32768.0,
                               (12, 10, 10), True, 1e-6, ntok, max_ctx)
        else:
            rmi.attn_prep_rope(q3, width, qn, kn, k, v, pos, qo, nh, nkv, hd, 64, 1e7, factor, 32768.0, 1e-6, ntok, max_ctx)
        outs.append([host(x).copy() for x in (qo, k, v)])
    (q0, k0, v0), (q1, k1, v1) = outs
    assert np.array_equal(q0.view(np.uint32), q1.view(np.uint32)) and np.array_equal(v0, v1)
    bits = [np.where(k.view(np.int16) < 0, -32768 - k.view(np.int16).astype(np.int32), k.view(np.int16)) for k in (k0, k1)]   # in order
    assert np.abs(bits[0] - bits[1]).max() <= 1 and (bits[0] != bits[1]).mean() < 0.01


@pytest.mark.parametrize("p0", [-1, 30, 2000000000])
def test_prep_axes_stores_nothing_outside_the_cache(rmi, p0):
    nh, nkv, hd, ntok, max_ctx = 2, 1, 128, 3, 32
    k, v = new_cache(rmi, ref.I8, max_ctx, nkv, hd), new_cache(rmi, ref.I4, max_ctx, nkv, hd)
    q3 = dev(np.ones((ntok, 2 * nh * hd + 2 * nkv * hd), np.float32))
    w, qo = dev(np.ones(hd, np.float32)), empty(ntok * nh * hd)
    kb, vb = host(k[0]).copy(), host(v[0]).copy()
    rmi.attn_prep_axes(q3, q3.shape[1], w, w, ref.I8, k[1], ref.I4, v[1], dev(np.array([p0], np.int32)), None, qo, nh, nkv, hd, 64, 1e4,
                       1.0, 0.0, (32, 0, 0), False, 1e-6, ntok, max_ctx)
    valid = {p for p in range(p0, p0 + ntok) if 0 <= p < max_ctx}
    assert changed_positions(kb[GUARD:-GUARD], host(k[1]), ref.I8, max_ctx, nkv, hd) <= valid
    assert changed_positions(vb[GUARD:-GUARD], host(v[1]), ref.I4, max_ctx, nkv, hd) <= valid
    assert np.array_equal(kb[:GUARD], host(k[0])[:GUARD]) and np.array_equal(vb[-GUARD:], host(v[0])[-GUARD:])


# ---- the accepted path ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n_kv,hd", [(4, 256), (3, 128)])
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("path,count", [([0], 1), ([2, 3, 7], 3), ([0, 1, 2, 5], 4), ([1, 2, 3, 4], 2), ([3, 2, 1, 0], 4), ([4, 4, 4], 3),
                                        (list(range(0, 64)), 64), (list(range(63, -1, -1)), 64), ([5, 6], 0), ([5, 6], -3), ([1, 2], 9)])
def test_compact(rmi, type_, n_kv, hd, path, count):
    rng = np.random.default_rng(8)
    max_ctx, base, caches = 90, 19, 3
    bufs = [new_cache(rmi, type_, max_ctx, n_kv, hd) for _ in range(caches)]
    before = []
    for whole, c in bufs:
        raw = rng.integers(0, 256, c.numel()).astype(np.uint8)
        c.copy_(torch().from_numpy(raw))
        before.append(raw)
    rmi.kv_compact(type_, [c for _, c in bufs], dev(np.array([base], np.int32)), dev(np.array(path, np.int32)),
                   dev(np.array([count], np.int32)), len(path), n_kv, hd, max_ctx)
    n = min(max(count, 0), len(path))
    for (whole, c), raw in zip(bufs, before):
        want = raw.copy()
        if type_ == ref.F16:
            parts = [(want.reshape(max_ctx, -1), raw.reshape(max_ctx, -1))]
        else:
            per = hd if type_ == ref.I8 else hd // 2
            cut = n_kv * max_ctx * per
            parts = []
            for lo, hi, w in ((0, cut, per), (cut, len(raw), hd // 32)):
                for h in range(n_kv):
                    parts.append(tuple(x[lo:hi].reshape(n_kv, max_ctx, w)[h] for x in (want, raw)))
        for dst, src in parts:
            for i in range(n):
                if base + path[i] < max_ctx:
                    dst[base + i] = src[base + path[i]]
        assert np.array_equal(host(c), want)
        assert (host(whole)[:GUARD] == 0x5a).all() and (host(whole)[-GUARD:] == 0x5a).all()


@pytest.mark.parametrize("base,path", [(-2, [1, 2, 3]), (30, [1, 5, 1]), (2000000000, [1]), (0, [-1, 40, 2])])
def test_compact_leaves_out_moves_outside_the_cache(rmi, base, path):
    max_ctx = 32
    whole, c = new_cache(rmi, ref.I8, max_ctx, 1, 128)
    raw = np.random.default_rng(9).integers(0, 256, c.numel()).astype(np.uint8)
    c.copy_(torch().from_numpy(raw))
    rmi.kv_compact(ref.I8, [c], dev(np.array([base], np.int32)), dev(np.array(path, np.int32)), dev(np.array([len(path)], np.int32)),
                   len(path), 1, 128, max_ctx)
    want = raw.copy()
    for i, p in enumerate(path):
        if 0 <= base + p < max_ctx and 0 <= base + i < max_ctx:
            for off, w in ((0, 128), (max_ctx * 128, 4)):
                want[off + (base + i) * w:off + (base + i + 1) * w] = raw[off + (base + p) * w:off + (base + p + 1) * w]
    assert np.array_equal(host(c), want)
    assert (host(whole)[:GUARD] == 0x5a).all() and (host(whole)[-GUARD:] == 0x5a).all()
