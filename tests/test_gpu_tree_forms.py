"""The forms of the tree attention (few rows, groups of 16, tiles of 32, 64 and 128 rows; one chunk, few, many) where a call meets
them only at particular sizes: what unwritten slots hold."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host, torch
from tests.test_gpu_tree_attn import Call

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
