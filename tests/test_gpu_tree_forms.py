"""The forms of the tree attention (few rows, groups of 16, tiles of 32, 64 and 128 rows; one chunk, few, many) where a call meets
them only at particular sizes: what unwritten slots hold, Q8_1 rows from every place that writes them, joins of many chunks, caches
longer than their text."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host, torch
from tests.test_gpu_tree_attn import Call, as_masks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


QUANT = [(ref.I8, ref.I8), (ref.I4, ref.I4), (ref.I8, ref.I4)]
QUANT_IDS = ["i8", "i4", "i8_i4"]
FIRST_ODD = {ref.I8: 199, ref.I4: 231}   # from this scale byte on s / 16 times 1152 or 72 passes fp16's largest number
# query heads, KV heads, dims, tokens, flag: 6, 12, 40 (groups, tiles of 64) and 80 rows (tiles of 128)
SHAPES = [(2, 2, 256, 6, 0), (1, 1, 128, 6, 0), (4, 2, 256, 6, 0), (2, 1, 128, 6, 0), (4, 2, 256, 20, 1), (4, 2, 256, 20, 0), (2, 1, 128, 20, 0),
          (2, 1, 128, 40, 0), (4, 2, 256, 40, 0)]


def put_row(raw, type_, max_ctx, nkv, hd, p, codes, sb):
    """code bytes and scale bytes of position p, every head"""
    per = hd if type_ == ref.I8 else hd // 2
    cut = nkv * max_ctx * per
    raw[:cut].reshape(nkv, max_ctx, per)[:, p] = codes[..., :per]
    raw[cut:].reshape(nkv, max_ctx, hd // 32)[:, p] = sb


@pytest.mark.parametrize("nh,nkv,hd,ntok,short", SHAPES)
@pytest.mark.parametrize("types", QUANT, ids=QUANT_IDS)
@pytest.mark.parametrize("kind", ["any", "high", "odd", "odd_v", "nan"])
def test_unseen_slots_hold_any_bytes(rmi, types, nh, nkv, hd, ntok, short, kind):
    """slot 2 of the draft holds bytes that no call wrote: nothing to the tokens whose masks leave it out"""
    base, rng = 70, np.random.default_rng(ntok + nh)
    sees = [t in (2, 3) or (t > 3 and t % 5 == 0) for t in range(ntok)]
    masks = [(1 << t) | (1 if t else 0) | (4 if sees[t] else 0) for t in range(ntok)]
    c = Call(rmi, types, nh, nkv, hd, ntok, base, masks, nsub=1 + short * rmi.TREE_SHORT)
    clean = c.run()
    for i, t in enumerate(types):
        lo, hi = {"any": (0, 256), "high": (ref.TOP[t] + 1, FIRST_ODD[t]), "odd": (FIRST_ODD[t], 255), "odd_v": (FIRST_ODD[t], 255), "nan": (255, 256)}[kind]
        if kind in ("high", "odd_v") and i == 0:
            continue   # K as it was
        c.raw[i] = c.raw[i].copy()
        codes = rng.integers(0, 256, (nkv, hd)).astype(np.uint8)
        if kind == "high":   # codes a quantiser writes: code + bias of 1 .. 2 bias - 1
            codes = rng.integers(1, 256, (nkv, hd)).astype(np.uint8) if t == ref.I8 else (rng.integers(1, 16, (nkv, hd)) * 17).astype(np.uint8)
        put_row(c.raw[i], t, c.max_ctx, nkv, hd, base + 2, codes, rng.integers(lo, hi, (nkv, hd // 32)).astype(np.uint8))
    y = c.run()
    for t in range(ntok):
        if not sees[t]:
            assert np.array_equal(y[t].view(np.uint32), clean[t].view(np.uint32)), f"token {t} does not see the slot"
    if kind in ("odd", "odd_v", "nan"):
        assert not np.isfinite(y[np.array(sees)]).any(), "a row that is seen is not left out"
    if kind == "high":
        want, bound = c.expected()
        assert (np.abs(y - want) <= bound).all()


@pytest.mark.parametrize("nh,nkv,hd,ntok,short", SHAPES)
def test_unseen_slots_of_fp16_hold_any_bits(rmi, nh, nkv, hd, ntok, short):
    base, rng = 70, np.random.default_rng(ntok + nh)
    masks = [(1 << t) | (1 if t else 0) | (4 if t in (2, 3) else 0) for t in range(ntok)]
    c = Call(rmi, (ref.F16, ref.F16), nh, nkv, hd, ntok, base, masks, nsub=1 + short * rmi.TREE_SHORT)
    clean = c.run()
    for i in range(2):
        c.raw[i] = c.raw[i].copy()
        c.raw[i].view(np.uint16).reshape(c.max_ctx, -1)[base + 2] = rng.integers(0, 1 << 16, nkv * hd)
    y = c.run()
    for t in range(ntok):
        if t not in (2, 3):
            assert np.array_equal(y[t].view(np.uint32), clean[t].view(np.uint32))


# a form's call: types, query heads, KV heads, dims, tokens, context, nsub, flag
PAIRS = [(ref.F16, ref.F16)] + QUANT
F16, I8, I4, I84 = PAIRS
FORMS = [
    # one chunk: the partial launch writes the result
    pytest.param(I8, 2, 2, 128, 1, 77, 1, 0, id="few8-one"), pytest.param(I4, 4, 2, 256, 6, 77, 1, 0, id="few16-one"),
    pytest.param(I84, 8, 2, 256, 11, 60, 1, 1, id="groups-one"), pytest.param(F16, 8, 2, 256, 7, 500, 6, 0, id="tile32-one"),
    pytest.param(F16, 8, 2, 128, 7, 500, 6, 0, id="tile32-128-one"), pytest.param(I8, 4, 2, 256, 20, 70, 1, 0, id="tile64-one"),
    pytest.param(I84, 2, 1, 128, 29, 70, 1, 0, id="tile64-128-one"), pytest.param(I4, 4, 2, 256, 40, 70, 1, 0, id="tile128-one"),
    pytest.param(F16, 8, 2, 128, 33, 70, 1, 0, id="tile128-128-one"),
    # two to eight chunks: the flat join
    pytest.param(I4, 4, 4, 256, 3, 300, 1, 0, id="few8-flat"), pytest.param(F16, 6, 2, 128, 5, 900, 1, 0, id="few16-flat"),
    pytest.param(I8, 8, 2, 256, 11, 400, 1, 1, id="groups-flat"), pytest.param(F16, 8, 2, 128, 7, 1600, 6, 0, id="tile32-128-flat"),
    pytest.param(I4, 4, 2, 128, 20, 300, 1, 0, id="tile64-flat"), pytest.param(I8, 8, 2, 256, 40, 300, 1, 0, id="tile128-flat"),
    # more chunks: the merge
    pytest.param(I8, 2, 2, 256, 2, 1300, 1, 0, id="few8-merge"), pytest.param(I84, 8, 4, 128, 6, 2500, 1, 0, id="few16-merge"),
    pytest.param(F16, 8, 2, 128, 9, 1500, 1, 1, id="groups-merge"), pytest.param(F16, 8, 2, 128, 7, 7000, 6, 0, id="tile32-128-merge"),
    pytest.param(F16, 4, 1, 256, 20, 1400, 1, 0, id="tile128-merge"), pytest.param(I4, 4, 2, 256, 17, 1500, 1, 0, id="tile64-merge"),
]


def form_call(rmi, types, nh, nkv, hd, ntok, base, nsub, short, masked=True, **kw):
    masks = ref.tree_masks(np.random.default_rng(ntok + base), ntok)[0] if masked else None
    return Call(rmi, types, nh, nkv, hd, ntok, base, masks, nsub=nsub + short * rmi.TREE_SHORT, seed=base, **kw)


@pytest.mark.parametrize("masked", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("types,nh,nkv,hd,ntok,base,nsub,short", FORMS)
def test_q8_rows_are_the_quantisers_of_y(rmi, orc, types, nh, nkv, hd, ntok, base, nsub, short, masked):
    """bytes, scale and sum: the quantiser's own of the fp32 rows, with y and without; the fp32 rows with Q8_1 and without"""
    c = form_call(rmi, types, nh, nkv, hd, ntok, base, nsub, short, masked)
    n = nh * hd
    for gate in (True, False):
        if not gate:
            c.q3 = None
        y, q8 = c.run(with_q8=True, pad=4)
        c.check(y)
        want = np.stack([orc.quantize_q8_1(y[t].reshape(-1), n) for t in range(ntok)])
        assert np.array_equal(q8[:, :n // 32 * 36], want) and (q8[:, n // 32 * 36:] == 0x33).all()
        assert np.array_equal(c.run().view(np.uint32), y.view(np.uint32))
        # Q8_1 alone
        alone = torch().full((ntok, n // 32 * 36), 0x33, dtype=torch().uint8, device="cuda:0")
        ws = empty(rmi.gqa_tree_workspace_bytes(c.max_ctx, nh, nkv, hd, ntok, c.nsub), "uint8")
        rmi.gqa_tree_decode(dev(c.q), types[0], dev(c.raw[0]), types[1], dev(c.raw[1]), dev(np.array([base], np.int32)), as_masks(c.masks),
                            dev(c.q3) if gate else None, c.width, None, 0, alone, n // 32 * 36, ws, nh, nkv, hd, ntok, c.max_ctx, c.nsub, c.scale)
        assert np.array_equal(host(alone), want)


@pytest.mark.parametrize("types,nh,nkv,hd,ntok,base,nsub,short", FORMS)
def test_a_cache_longer_than_its_text(rmi, types, nh, nkv, hd, ntok, base, nsub, short):
    """positions past the draft are nothing to anyone, whichever join their number of chunks takes; their records are not read (the
    workspace holds NaN before)"""
    for more in (3 * 128 * nsub, 40 * 128 * nsub):
        c = form_call(rmi, types, nh, nkv, hd, ntok, base, nsub, short, max_ctx=base + ntok + more)
        for raw, t in zip(c.raw, types):
            if t == ref.F16:
                raw.view(np.uint16).reshape(c.max_ctx, -1)[base + ntok:] = 0x7e00
            else:
                raw[nkv * c.max_ctx * (hd if t == ref.I8 else hd // 2):].reshape(nkv, c.max_ctx, -1)[:, base + ntok:] = 255
        with np.errstate(invalid="ignore"):
            c.check()


@pytest.mark.parametrize("chunks", [65, 130, 300])
@pytest.mark.parametrize("types,nh,ntok,short", [(I8, 1, 2, 0), (I4, 4, 3, 0), (F16, 4, 1, 0), (I84, 4, 6, 1), (F16, 8, 9, 0)])
def test_joins_of_many_chunks(rmi, types, nh, ntok, short, chunks):
    """more chunks than the merge takes at a time (64 outputs in flight, a weight a lane)"""
    c = form_call(rmi, types, nh, 1, 128, ntok, 128 * chunks - ntok, 1, short, max_ctx=128 * chunks)
    c.check()
    c.masks = None
    c.check()


def test_as_many_chunks_as_there_may_be(rmi):
    c = form_call(rmi, F16, 2, 1, 128, 1, 128 * 2048 - 1, 1, 0, False, max_ctx=128 * 2048)
    c.check()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("nh,nkv,ntok,base,nsub", [(8, 2, 5, 0, 6), (8, 2, 8, 760, 6), (4, 4, 17, 300, 7), (32, 2, 2, 2000, 6), (6, 1, 5, 1535, 6),
                                                   (2, 2, 32, 769, 6)])
def test_fp16_tiles_of_32_rows(rmi, nh, nkv, ntok, base, nsub, hd):
    for masked in (True, False):
        form_call(rmi, F16, nh, nkv, hd, ntok, base, nsub, 0, masked).check()


@pytest.mark.parametrize("ntok,used", [(1, 448), (6, 512), (20, 448), (40, 441)])
def test_an_fp16_cache_by_the_positions_in_use(rmi, ntok, used):
    """its layout does not hang on max_ctx: a call may be given the part that holds the text"""
    c = form_call(rmi, F16, 4, 2, 256, ntok, 401, 1, 0, max_ctx=5000)
    c.check()
    k, v = c.values()
    c.max_ctx = used   # of the same buffers
    c.values = lambda: (k[:used], v[:used])
    c.check()


@pytest.mark.parametrize("nh,nkv,hd,ntok,short", SHAPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_an_infinity_in_a_key_that_is_seen(rmi, nh, nkv, hd, ntok, short, bad):
    """in one dim of a row of the context: NaN, or the formula's result; where that is NaN (a score of infinity), NaN"""
    base, rng = 70, np.random.default_rng(4)
    kv = [rng.standard_normal((base + ntok + 5, nkv, hd)).astype(np.float32) for _ in range(2)]
    kv[0][30, :, 7] = bad
    c = Call(rmi, (ref.F16, ref.F16), nh, nkv, hd, ntok, base, None, nsub=1 + short * rmi.TREE_SHORT, kv=kv)
    y = c.run()
    with np.errstate(all="ignore"):
        want, _ = c.expected()
        c.raw[0] = c.raw[0].copy()
        c.raw[0].view(np.float16).reshape(c.max_ctx, nkv, hd)[30, :, 7] = 0   # a bound without the infinity
        bound = c.expected()[1]
    nan = np.isnan(y).all(-1)
    assert (nan | ~np.isnan(y).any(-1)).all() and nan[np.isnan(want).any(-1)].all()
    assert (np.abs(y - want) <= bound)[~nan].all()
