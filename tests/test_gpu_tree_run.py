"""The quantised-cache operators as a serving loop uses them: a prompt ingested, then rounds of a drafted tree (norm, rotation and
cache write at the nodes' depths, attention by ancestor masks, logits of every node processed, argmax, the accepted path's rows
moved), next to the same tokens decoded one by one; then the round as a captured graph."""
import numpy as np
import pytest

from tests import kv_ref as ref
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu

NH, NKV, HD, NROT, VOCAB, CTX, PROMPT, NODES, LAYERS = 8, 2, 128, 64, 777, 256, 133, 12, 2
WIDTH = 2 * NH * HD + 2 * NKV * HD
SECTIONS = (12, 10, 10)
SCALE = HD ** -0.5
PAIRS = [(ref.F16, ref.F16), (ref.I8, ref.I8), (ref.I4, ref.I4), (ref.I8, ref.I4)]
IDS = ["f16", "i8", "i4", "i8_i4"]


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


class Text:
    """The caches of one text, and the calls on them.  A token's q / k / v depend on its id alone (the layers' tables), so two
    texts with the same tokens hold the same rows."""

    def __init__(self, rmi, types, seed=5):
        rng = np.random.default_rng(seed)
        self.rmi, self.types = rmi, types
        self.tables = [dev(rng.standard_normal((VOCAB, WIDTH)).astype(np.float32)) for _ in range(LAYERS)]
        self.qn = [dev((1 + 0.1 * rng.standard_normal(HD)).astype(np.float32)) for _ in range(LAYERS)]
        self.kn = [dev((1 + 0.1 * rng.standard_normal(HD)).astype(np.float32)) for _ in range(LAYERS)]
        self.head = dev(rng.standard_normal((VOCAB, VOCAB)).astype(np.float32))
        self.caches = [[torch().zeros(rmi.kv_cache_bytes(t, CTX, NKV, HD), dtype=torch().uint8, device="cuda:0") for t in types]
                       for _ in range(LAYERS)]
        self.pos = dev(np.zeros(1, np.int32))

    def forward(self, ids, axis_pos=None, masks=None, nsub=1):
        """per layer q and y of the tokens `ids` (device), whose rows go to the slots from pos on"""
        n, rmi, out = len(ids), self.rmi, []
        ws = empty(rmi.gqa_tree_workspace_bytes(CTX, NH, NKV, HD, n, nsub), "uint8")
        for l in range(LAYERS):
            q3 = self.tables[l][ids]
            q, y = empty(n * NH * HD), empty(n * NH * HD)
            k, v = self.caches[l]
            rmi.attn_prep_axes(q3, WIDTH, self.qn[l], self.kn[l], self.types[0], k, self.types[1], v, self.pos, axis_pos, q, NH, NKV, HD,
                               NROT, 1e6, 1.0, 0.0, SECTIONS, True, 1e-6, n, CTX)
            rmi.gqa_tree_decode(q, self.types[0], k, self.types[1], v, self.pos, masks, q3, WIDTH, y, NH * HD, None, 0, ws, NH, NKV, HD, n,
                                CTX, nsub, SCALE)
            out.append((q3, q, y))
        return out

    def logits(self, y, history, length, draft, masks, allow):
        n = len(draft)
        x = self.head[draft.long()] + y.view(n, NH * HD)[:, :VOCAB]   # stands for the output product
        z, idx = empty(n * VOCAB), empty(n, "int32")
        self.rmi.logits_process(x, VOCAB, n, VOCAB, z, VOCAB, history, length, CTX, 50, draft, masks, n, 1.3, 0.25, 0.5, allow=allow,
                                allow_stride=(VOCAB + 31) // 32)
        self.rmi.argmax(z, VOCAB, idx, empty(self.rmi.argmax_workspace_bytes(n), "uint8"), n, VOCAB)
        return x, z, idx

    def accept(self, path, count):
        for i in (0, 1):
            self.rmi.kv_compact(self.types[i], [c[i] for c in self.caches], self.pos, path, count, NODES, NKV, HD, CTX)

    def rows(self, n):
        """positions [0, n) of every cache, read back"""
        out = []
        for c in self.caches:
            for i in (0, 1):
                t = empty(CTX * NKV * HD)
                self.rmi.kv_read(self.types[i], c[i], t, NKV * HD, 0, n, NKV, HD, CTX)
                out.append(host(t)[:n * NKV * HD])
        return out

    def check(self, out, base, n, masks):
        """the layers' y against softmax attention in 64 bits over what the caches hold"""
        for (q3, q, y), c in zip(out, self.caches):
            k, v = (ref.decode(host(r), t, CTX, NKV, HD) for r, t in zip(c, self.types))
            gate = host(q3)[:, :2 * NH * HD].reshape(n, NH, 2, HD)[:, :, 1].astype(np.float64)
            want, bound = ref.attention(host(q).reshape(n, NH, HD).astype(np.float64), k, v, base, masks, np.float64(np.float32(SCALE)), gate)
            assert (np.abs(host(y).reshape(n, NH, HD) - want) <= bound).all()


def draw_round(rng, base):
    """a tree's ids, masks and axis positions, a grammar, and the path to one of its nodes"""
    masks, depth = ref.tree_masks(rng, NODES, reach=4)
    ids = rng.integers(0, VOCAB, NODES)
    allow = rng.integers(0, 2 ** 32, (NODES, (VOCAB + 31) // 32), dtype=np.uint32)
    leaf = int(rng.integers(NODES // 2, NODES))
    path = [j for j in range(NODES) if masks[leaf] >> j & 1]
    axes = np.tile(base + np.array(depth, np.int32), (3, 1)).astype(np.int32)
    return masks, ids, axes, allow, path


def device(masks, ids, axes, allow, path):
    return (dev(np.array(masks, np.uint64).view(np.int64)), dev(ids.astype(np.int64)), dev(ids.astype(np.int32)), dev(axes),
            dev(allow.view(np.int32)), dev(np.array(path + [0] * (NODES - len(path)), np.int32)), dev(np.array([len(path)], np.int32)))


def history_of(ids):
    return dev(np.concatenate([ids, np.full(CTX - len(ids), -1)]).astype(np.int32)), dev(np.array([len(ids)], np.int32))


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
def test_rounds_of_trees_hold_what_single_tokens_hold(rmi, types):
    rng = np.random.default_rng(types[0] * 3 + types[1])
    trees, single = Text(rmi, types), Text(rmi, types)
    text = [int(i) for i in rng.integers(0, VOCAB, PROMPT)]
    for t in (trees, single):
        out = t.forward(dev(np.array(text, np.int64)))
        t.pos.fill_(PROMPT)
    trees.check(out, 0, PROMPT, None)
    for _ in range(3):
        base = len(text)
        masks, ids, axes, allow, path = draw_round(rng, base)
        dm, d64, d32, dax, dal, dpath, dcount = device(masks, ids, axes, allow, path)
        out = trees.forward(d64, dax, dm)
        trees.check(out, base, NODES, masks)
        x, z, idx = trees.logits(out[-1][2], *history_of(text), d32, dm, dal)
        xh, zh = host(x), host(z).reshape(NODES, VOCAB)
        want = ref.logits(xh, text, 50, [int(i) for i in ids], masks, 1.3, 0.25, 0.5, [], [], allow)
        fin = np.isfinite(want)
        assert np.array_equal(np.isfinite(zh), fin)
        # the repetition factor's rounding to fp32, the product's, the sum's and the difference's: 2^-24 each of at most
        # |x| 1.3 + 50 * 0.5 + 0.25
        assert (np.abs(zh[fin] - want[fin]) <= 4 * 2.0 ** -24 * (np.abs(xh[fin]) * 1.3 + 25.25)).all()
        assert np.array_equal(host(idx), zh.argmax(1))
        trees.accept(dpath, dcount)
        trees.pos += len(path)
        for i in path:
            last = single.forward(dev(np.array([ids[i]], np.int64)))
            single.pos += 1
        text += [int(ids[i]) for i in path]
        for a, b in zip(trees.rows(len(text)), single.rows(len(text))):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
        # the accepted leaf's result: the same rows seen in another order, so within both sides' bounds
        for (_, _, y), (q3, q, y1), c in zip(out, last, single.caches):
            k, v = (ref.decode(host(r), t, CTX, NKV, HD) for r, t in zip(c, types))
            _, bound = ref.attention(host(q).reshape(1, NH, HD).astype(np.float64), k, v, len(text) - 1, None, SCALE)
            assert (np.abs(host(y).reshape(NODES, NH, HD)[path[-1]] - host(y1).reshape(1, NH, HD)[0]) <= 2 * bound[0]).all()
    # one more token behind the moved rows: the same bits
    for (_, _, a), (_, _, b) in zip(trees.forward(dev(np.array([3], np.int64))), single.forward(dev(np.array([3], np.int64)))):
        assert np.array_equal(host(a).view(np.uint32), host(b).view(np.uint32))


@pytest.mark.parametrize("types", PAIRS, ids=IDS)
def test_a_captured_round_replays(rmi, types):
    """the whole round in one graph, on a stream of its own; its inputs change between replays, eager rounds run between them"""
    t = torch()
    rng = np.random.default_rng(9)
    eager, graph = Text(rmi, types), Text(rmi, types)
    text = [int(i) for i in rng.integers(0, VOCAB, PROMPT)]
    for x in (eager, graph):
        x.forward(dev(np.array(text, np.int64)))
        x.pos.fill_(PROMPT)
    bufs = device(*draw_round(rng, PROMPT))
    hist, length = history_of(text)

    def step(x, dm, d64, d32, dax, dal, dpath, dcount):
        out = x.forward(d64, dax, dm)
        res = x.logits(out[-1][2], hist, length, d32, dm, dal)
        x.accept(dpath, dcount)
        x.pos += dcount
        return [y for _, _, y in out] + list(res)

    keep = [c.clone() for l in graph.caches for c in l]
    step(graph, *bufs)   # first use of every kernel
    t.cuda.synchronize()
    for c, k in zip((c for l in graph.caches for c in l), keep):
        c.copy_(k)
    graph.pos.fill_(PROMPT)
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=t.cuda.Stream()):
        got = step(graph, *bufs)
    for _ in range(4):
        base = len(text)
        masks, ids, axes, allow, path = draw_round(rng, base)
        for b, x in zip(bufs, device(masks, ids, axes, allow, path)):
            b.copy_(x)
        h, n = history_of(text)
        hist.copy_(h)
        length.copy_(n)
        t.cuda.synchronize()
        g.replay()
        t.cuda.synchronize()
        want = step(eager, *bufs)
        t.cuda.synchronize()
        for a, b in zip(got, want):
            assert np.array_equal(host(a).view(np.uint32), host(b).view(np.uint32))
        text += [int(ids[i]) for i in path]
        assert int(host(graph.pos)[0]) == len(text) == int(host(eager.pos)[0])
        for a, b in zip(graph.rows(len(text)), eager.rows(len(text))):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_two_calls_at_once(rmi):
    """two streams, a workspace each, the same caches: each call's bits are those of the call alone"""
    t = torch()
    rng = np.random.default_rng(1)
    nkv, nh, hd, ctx, n = 4, 16, 256, 6000, 8
    caches = [dev(ref.encode(rng.standard_normal((ctx, nkv, hd)).astype(np.float32), ref.I8)) for _ in range(2)]
    masks = [dev(np.array(ref.tree_masks(rng, n)[0], np.uint64).view(np.int64)) for _ in range(2)]
    qs = [dev(rng.standard_normal((n, nh, hd)).astype(np.float32)) for _ in range(2)]
    pos = [dev(np.array([p], np.int32)) for p in (ctx - n, 2500)]
    nsub = rmi.gqa_tree_nsub(ctx, nh, nkv, hd, n)
    need = rmi.gqa_tree_workspace_bytes(ctx, nh, nkv, hd, n, nsub)
    ws, ys, streams = [empty(need, "uint8") for _ in range(2)], [empty(n * nh * hd) for _ in range(2)], [t.cuda.Stream() for _ in range(2)]

    def call(i, stream):
        rmi.gqa_tree_decode(qs[i], ref.I8, caches[0], ref.I8, caches[1], pos[i], masks[i], None, 0, ys[i], nh * hd, None, 0, ws[i], nh, nkv,
                            hd, n, ctx, nsub, hd ** -0.5, stream=stream)

    want = []
    for i in range(2):
        call(i, None)
        want.append(host(ys[i]).copy())
        ys[i].zero_()
    t.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            call(i, streams[i])
    t.cuda.synchronize()
    for i in range(2):
        assert np.array_equal(host(ys[i]).view(np.uint32), want[i].view(np.uint32))


@pytest.mark.parametrize("type_,ntok", [(ref.F16, 3), (ref.F16, 70), (ref.I8, 3), (ref.I8, 40), (ref.I4, 5)])
def test_a_cache_beyond_32_bit_offsets(rmi, type_, ntok):
    """2.3 million positions x 8 heads x 256: rows at the far end written, seen, moved and read back; the others are zero, so the
    softmax has a closed form"""
    t = torch()
    nkv, hd, ctx = 8, 256, 2300000
    rng = np.random.default_rng(ntok)
    caches = [t.zeros(rmi.kv_cache_bytes(type_, ctx, nkv, hd), dtype=t.uint8, device="cuda:0") for _ in range(2)]
    n, base = ntok + 4, ctx - ntok          # four rows of the context, then the draft, which ends with the cache
    rows = [rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2)]
    for c, x in zip(caches, rows):
        rmi.kv_write(type_, dev(x), nkv * hd, c, base - 4, n, nkv, hd, ctx)
    held = [ref.held(x, type_) for x in rows]
    q = rng.standard_normal((ntok, nkv, hd)).astype(np.float32)
    pos = dev(np.array([base], np.int32))
    nsub = rmi.gqa_tree_nsub(ctx, nkv, nkv, hd, ntok)
    ws, y = empty(rmi.gqa_tree_workspace_bytes(ctx, nkv, nkv, hd, ntok, nsub), "uint8"), empty(ntok * nkv * hd)
    scale = 0.75   # scores of about +-12: the few rows weigh as much as the zeros
    rmi.gqa_tree_decode(dev(q), type_, caches[0], type_, caches[1], pos, None, None, 0, y, nkv * hd, None, 0, ws, nkv, nkv, hd, ntok, ctx, nsub,
                        scale)
    got = host(y).reshape(ntok, nkv, hd)
    for i in range(ntok):
        m = 4 + i + 1
        s = np.einsum("hd,phd->hp", q[i].astype(np.float64), held[0][:m]) * scale
        top = np.maximum(s.max(1, keepdims=True), 0)
        w = np.exp(s - top)
        total = w.sum(1) + (base - 4) * np.exp(-top[:, 0])
        want = np.einsum("hp,phd->hd", w, held[1][:m]) / total[:, None]
        # a weight's relative error: its score's ((hd + 8) roundings of the sum of |q k|), the exponent's and the sum's (a lane
        # adds once per step of 32 positions, a chunk's wave has nsub of them)
        a = np.einsum("hd,phd->hp", np.abs(q[i]).astype(np.float64), np.abs(held[0][:m])).max(1) * scale
        rel = 2 * (hd + 8) * 2.0 ** -24 * a + 2.0 ** -18 + (m + (nsub & (rmi.TREE_SHORT - 1))) * 2.0 ** -24
        assert (np.abs(got[i] - want) <= (rel * (w @ np.ones(m)) / total * np.abs(held[1]).max())[:, None]).all()
    path = [1, ntok - 1]
    rmi.kv_compact(type_, caches, pos, dev(np.array(path, np.int32)), dev(np.array([2], np.int32)), 2, nkv, hd, ctx)
    out = empty(n * nkv * hd)
    for c, h in zip(caches, held):
        rmi.kv_read(type_, c, out, nkv * hd, base - 4, n, nkv, hd, ctx)
        want = h.copy()
        want[4], want[5] = h[4 + path[0]], h[4 + path[1]]
        assert np.array_equal(host(out).reshape(n, nkv, hd).astype(np.float64), want)
    del caches
    t.cuda.empty_cache()
