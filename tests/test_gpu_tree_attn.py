"""Attention of drafted trees and chains over 16-, 8- and 4-bit caches, against softmax attention in 64 bits over the values
the cache holds (tests/kv_ref.py).  The bar is an fp32 error bound computed from the inputs (kv_ref.attention)."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu

PAIRS = [(ref.F16, ref.F16), (ref.I8, ref.I8), (ref.I4, ref.I4), (ref.I8, ref.I4)]
IDS = ["f16", "i8", "i4", "i8_i4"]


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def as_masks(masks):
    return None if masks is None else dev(np.array(masks, np.uint64).view(np.int64))


class Call:
    """inputs of one call, in host memory, and the call itself"""

    def __init__(self, rmi, types, nh, nkv, hd, ntok, base, masks, max_ctx=None, nsub=None, seed=1, gate=True, kv=None):
        rng = np.random.default_rng(seed)
        self.rmi, self.types, self.nh, self.nkv, self.hd, self.ntok, self.base, self.masks = rmi, types, nh, nkv, hd, ntok, base, masks
        self.max_ctx = max_ctx or base + ntok + 5
        self.q = rng.standard_normal((ntok, nh, hd)).astype(np.float32)
        if kv is None:
            kv = [rng.standard_normal((self.max_ctx, nkv, hd)).astype(np.float32) for _ in range(2)]
        self.raw = [ref.encode(x, t) for x, t in zip(kv, types)]
        self.width = 2 * nh * hd + 2 * nkv * hd
        self.q3 = rng.standard_normal((ntok, self.width)).astype(np.float32) if gate else None
        self.scale = hd ** -0.5
        self.nsub = nsub or rmi.gqa_tree_nsub(base + ntok, nh, nkv, hd, ntok)

    def values(self):
        return [ref.decode(r, t, self.max_ctx, self.nkv, self.hd) for r, t in zip(self.raw, self.types)]

    def run(self, with_q8=False, tokens=None, base=None, masks="own", pad=0):
        """y [ntok, nh, hd]; tokens: the slice of the query tokens that is sent, base: another pos[0]"""
        q = self.q if tokens is None else self.q[tokens]
        q3 = None if self.q3 is None else self.q3 if tokens is None else self.q3[tokens]
        n = len(q)
        masks = self.masks if isinstance(masks, str) else masks
        need = self.rmi.gqa_tree_workspace_bytes(self.max_ctx, self.nh, self.nkv, self.hd, n, self.nsub)
        ws = torch().full((need + 64,), 0xff, dtype=torch().uint8, device="cuda:0")   # NaN records where nothing is written
        yw, qw = self.nh * self.hd + pad, self.nh * self.hd // 32 * 36 + 4 * pad
        y = torch().full((n, yw), 7.0, device="cuda:0")
        q8 = torch().full((n, qw), 0x33, dtype=torch().uint8, device="cuda:0") if with_q8 else None
        self.rmi.gqa_tree_decode(dev(q), self.types[0], dev(self.raw[0]), self.types[1], dev(self.raw[1]),
                                 dev(np.array([self.base if base is None else base], np.int32)), as_masks(masks),
                                 None if q3 is None else dev(q3), self.width, y, yw, q8, qw, ws, self.nh, self.nkv, self.hd, n, self.max_ctx,
                                 self.nsub, self.scale)
        yh = host(y)
        assert (yh[:, self.nh * self.hd:] == 7.0).all()
        assert (host(ws)[need:] == 0xff).all(), "the workspace is longer than it says"
        out = yh[:, :self.nh * self.hd].reshape(n, self.nh, self.hd)
        return (out, host(q8)) if with_q8 else out

    def expected(self):
        k, v = self.values()
        gate = None if self.q3 is None else self.q3[:, :2 * self.nh * self.hd].reshape(self.ntok, self.nh, 2, self.hd)[:, :, 1].astype(np.float64)
        with np.errstate(invalid="ignore"):
            return ref.attention(self.q.astype(np.float64), k, v, self.base, self.masks, np.float64(np.float32(self.scale)), gate)

    def check(self, y=None):
        want, bound = self.expected()
        got = self.run() if y is None else y
        err = np.abs(got - want)
        assert (err <= bound).all(), f"error {err.max():.3e} of {np.abs(want).max():.3e}, {(err / np.maximum(bound, 1e-30)).max():.2f} of the bound"
        return got


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 4, 256), (8, 2, 128), (2, 2, 256), (5, 1, 128), (6, 2, 256), (24, 1, 128)])
@pytest.mark.parametrize("ntok,base", [(1, 0), (1, 1), (2, 31), (3, 127), (8, 128), (5, 300)])
def test_trees(rmi, types, nh, nkv, hd, ntok, base):
    masks, _ = ref.tree_masks(np.random.default_rng(ntok * 1000 + base), ntok)
    Call(rmi, types, nh, nkv, hd, ntok, base, masks, seed=base + ntok).check()


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
@pytest.mark.parametrize("ntok,base,nsub", [(5, 1700, 6), (8, 1500, 7), (1, 0, 1), (1, 999, 1), (2, 1023, 2), (7, 255, 1), (33, 100, 1), (64, 64, 3), (65, 0, 1), (130, 515, 2)])
def test_chains(rmi, types, ntok, base, nsub):
    Call(rmi, types, 8, 2, 256, ntok, base, None, seed=ntok, nsub=nsub).check()


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
@pytest.mark.parametrize("ntok,base,nsub,masked", [(5, 1700, 6, True), (5, 200, 1, False), (17, 0, 1, True), (33, 700, 2, True), (64, 1100, 3, True),
                                                   (64, 3, 9, True), (130, 515, 2, False), (300, 1, 1, False)])
def test_groups_of_sixteen_rows(rmi, types, ntok, base, nsub, masked):
    masks = ref.tree_masks(np.random.default_rng(ntok), ntok, reach=9)[0] if masked else None
    Call(rmi, types, 8, 2, 128 if ntok % 2 else 256, ntok, base, masks, seed=ntok, nsub=nsub + rmi.TREE_SHORT).check()


@pytest.mark.parametrize("ntok", [17, 40, 64])
@pytest.mark.parametrize("types", PAIRS, ids=IDS)
def test_wide_trees_over_many_chunks(rmi, types, ntok):
    masks, _ = ref.tree_masks(np.random.default_rng(ntok), ntok, reach=9)
    Call(rmi, types, 8, 4, 128, ntok, 700, masks, seed=ntok, nsub=1).check()


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
def test_nothing_seen_gives_zeros(rmi, types):
    """tokens without a context whose mask is empty, next to tokens that see themselves or others"""
    c = Call(rmi, types, 4, 2, 256, 5, 0, [0, 2, 0, 0b01010, 0b10001])
    y = c.check()
    assert not y[0].any() and not y[2].any() and y[1].any()


def test_mask_bits_without_a_token_are_ignored(rmi):
    c = Call(rmi, (ref.F16, ref.F16), 4, 2, 256, 3, 70, [1, 3, 5])
    want = c.check()
    assert np.array_equal(c.run(masks=[m | 0xfffffffffffffff8 for m in (1, 3, 5)]), want)


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("what", ["k", "v", "both"])
def test_unseen_rows_hold_anything(rmi, types, bad, what):
    """a branch whose K / V rows are not finite is nothing to the others, and rows past the draft are nothing to anyone"""
    base, ntok, hd, nkv = 90, 6, 256, 2
    masks = [1, 3, 4, 12, 0b10001, 0b100100]    # token 2's rows are bad: only tokens 2, 3 and 5 see them
    rng = np.random.default_rng(3)
    kv = [rng.standard_normal((base + ntok + 30, nkv, hd)).astype(np.float32) for _ in range(2)]
    clean = Call(rmi, types, 4, nkv, hd, ntok, base, masks, max_ctx=base + ntok + 30, kv=kv, nsub=1)
    for i, x in enumerate(kv):
        if what in ("kv"[i], "both"):
            x[base + 2, :, 5::7] = bad
            x[base + ntok:] = bad
    c = Call(rmi, types, 4, nkv, hd, ntok, base, masks, max_ctx=base + ntok + 30, kv=kv, nsub=1)
    y, z = c.run(), clean.run()
    for t in (0, 1, 4):
        assert np.isfinite(y[t]).all()
        assert np.array_equal(y[t], z[t])
    with np.errstate(all="ignore"):
        want, bound = c.expected()
    for t in (2, 3, 5):   # what does see them gets what the formula gives
        assert np.array_equal(np.isfinite(y[t]), np.isfinite(want[t]))
        fin = np.isfinite(want[t])
        assert np.array_equal(np.isnan(y[t])[~fin], np.isnan(want[t])[~fin])
        assert np.array_equal(y[t][~fin & ~np.isnan(want[t])], want[t][~fin & ~np.isnan(want[t])])


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
@pytest.mark.parametrize("ntok", [1, 3, 6, 20, 40])
def test_a_result_that_is_not_a_number_is_not_zero(rmi, types, ntok):
    """a NaN in q, or scores of a row that are all NaN or -infinity, is no row that sees nothing"""
    masks = [1 << i for i in range(ntok)]
    masks[0] |= 2 if ntok == 3 else 0
    c = Call(rmi, types, 8, 2, 256, ntok, 0, masks, nsub=1)
    for m in (masks, None):
        c.masks = m
        for what in ("q", "k", "-inf"):
            q, raw = c.q.copy(), c.raw
            c.q, t = np.abs(c.q) + 0.5, ntok - 1
            if what == "q":
                c.q[t, 3, 17] = np.nan
            else:   # the rows of the last token: with masks it sees them alone
                k = c.values()[0].astype(np.float32)
                k[:ntok, :, :] = np.nan if what == "k" else -np.inf
                c.raw = [ref.encode(k, types[0]), raw[1]]
            y = c.run()
            c.q, c.raw = q, raw
            assert np.isnan(y[t, 3]).all()
            if what == "q":
                assert np.isfinite(np.delete(y, 3, 1)).all() and np.isfinite(y[:t, 3]).all()


@pytest.mark.parametrize("types", PAIRS[1:], ids=IDS[1:])
@pytest.mark.parametrize("ntok,base", [(1, 700), (6, 333), (40, 500)])
def test_quantised_caches_give_the_bits_of_an_fp16_cache_of_their_values(rmi, types, ntok, base):
    masks, _ = ref.tree_masks(np.random.default_rng(2), ntok)
    c = Call(rmi, types, 16, 4, 256, ntok, base, masks, nsub=1)
    raw = c.raw
    for nsub in (1, 2 + rmi.TREE_SHORT):
        c.types, c.raw, c.nsub = types, raw, nsub
        y = c.run()
        c.raw = [ref.encode(x, ref.F16) for x in c.values()]
        c.types = (ref.F16, ref.F16)
        assert np.array_equal(y.view(np.uint32), c.run().view(np.uint32))


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
def test_a_chain_by_masks_is_a_chain(rmi, types):
    n = 20
    c = Call(rmi, types, 8, 2, 128, n, 250, [(2 << i) - 1 for i in range(n)], nsub=1)
    assert np.array_equal(c.run().view(np.uint32), c.run(masks=None).view(np.uint32))


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
@pytest.mark.parametrize("nh,ntok", [(16, 2), (8, 4), (4, 8), (4, 3)])
def test_a_short_chains_tokens_are_the_single_tokens(rmi, types, nh, ntok):
    """up to 8 query rows per KV head: every token of a chain has the bits of a decode step at its slot"""
    c = Call(rmi, types, nh, 4, 256, ntok, 381, None, nsub=2)
    y = c.run()
    for t in range(ntok):
        one = c.run(tokens=slice(t, t + 1), base=c.base + t)
        assert np.array_equal(one[0].view(np.uint32), y[t].view(np.uint32))


def test_same_inputs_same_bits(rmi):
    masks, _ = ref.tree_masks(np.random.default_rng(4), 30)
    c = Call(rmi, (ref.I8, ref.I4), 16, 4, 256, 30, 900, masks)
    assert np.array_equal(c.run().view(np.uint32), c.run().view(np.uint32))


@pytest.mark.parametrize("hd", [128, 256])
def test_q8_output_gate_and_strides(rmi, orc, hd):
    c = Call(rmi, (ref.I8, ref.I8), 4, 2, hd, 6, 77, ref.tree_masks(np.random.default_rng(5), 6)[0])
    y, q8 = c.run(with_q8=True, pad=4)
    c.check(y)
    n = 4 * hd
    assert (q8[:, n // 32 * 36:] == 0x33).all()
    deq = np.stack([orc.dequantize_q8_1(np.ascontiguousarray(r[:n // 32 * 36]), n) for r in q8]).reshape(6, -1, 32).astype(np.float64)
    r = y.reshape(6, -1, 32).astype(np.float64)
    # half a step of amax / 127, and the fp16 rounding (2^-11) of the step at up to 127 steps
    assert (np.abs(deq - r) <= np.abs(r).max(-1, keepdims=True) * (0.5 / 127 + 2.0 ** -11) * (1 + 1e-6)).all()
    c.q3 = None
    c.check()
    # y alone, q8 alone
    c2 = Call(rmi, (ref.I8, ref.I8), 4, 2, hd, 1, 5, None)
    a, b = c2.run(with_q8=True)
    assert np.array_equal(a, c2.run())


@pytest.mark.parametrize("base", [-1, 62, 64, 2000000000])
def test_a_draft_outside_the_cache_writes_nothing(rmi, base):
    c = Call(rmi, (ref.F16, ref.F16), 4, 2, 128, 3, 10, None, max_ctx=64, nsub=1)
    assert (c.run(base=base) == 7.0).all()


@pytest.mark.parametrize("base", [61, 0])
def test_a_draft_at_the_ends_of_the_cache(rmi, base):
    c = Call(rmi, (ref.I4, ref.I4), 4, 2, 128, 3, base, None, max_ctx=64, nsub=1)
    c.check()


def test_large_scores(rmi):
    """scores of a few hundred: one position holds the weight, the others underflow"""
    c = Call(rmi, (ref.F16, ref.F16), 4, 2, 256, 4, 500, [1, 3, 5, 9], nsub=1)
    c.q *= 60
    y, (want, bound) = c.run(), c.expected()
    # the weights' error grows with the score's: |s| < 2^9 takes the exponent's share to 2^-15
    assert (np.abs(y - want) <= bound + 2.0 ** -15 * 4).all()


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
def test_graph_replays(rmi, types):
    """captured once, replayed behind a context that grows: the position is read on the device"""
    t = torch()
    c = Call(rmi, types, 8, 2, 256, 4, 100, ref.tree_masks(np.random.default_rng(6), 4)[0], max_ctx=512, nsub=1)
    q, k, v, pos, masks, q3 = dev(c.q), dev(c.raw[0]), dev(c.raw[1]), dev(np.array([100], np.int32)), as_masks(c.masks), dev(c.q3)
    ws = empty(rmi.gqa_tree_workspace_bytes(512, 8, 2, 256, 4, 1), "uint8")
    y = empty(4 * 8 * 256)

    def step():
        rmi.gqa_tree_decode(q, types[0], k, types[1], v, pos, masks, q3, c.width, y, 8 * 256, None, 0, ws, 8, 2, 256, 4, 512, 1, c.scale)

    step()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=t.cuda.Stream()):
        step()
    for base in (100, 3, 350, 0, 508):
        pos.fill_(base)
        ws.fill_(0xff)
        g.replay()
        t.cuda.synchronize()
        c.base = base
        c.check(host(y).reshape(4, 8, 256))
