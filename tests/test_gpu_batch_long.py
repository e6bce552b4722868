"""Attention of a batch at lengths where a lost step or chunk would be small: every position counted, every key found, and the formula
in 64 bits with a bound that follows the data (tests/batch_exact.py)."""
import numpy as np
import pytest

from . import batch_exact as exact
from . import batch_ref as ref
from . import kv_ref
from .gpu_util import torch
from .test_gpu_batch_attn import TYPES, Batch, ints

pytestmark = pytest.mark.gpu
F16, I8, I4 = kv_ref.F16, kv_ref.I8, kv_ref.I4


@pytest.fixture(scope="module")
def rmi():
    torch()
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


class Given(Batch):
    """a batch whose K and V rows are given, [positions, n_kv, hd] of each request; two rows of padding"""

    def __init__(self, rng, lens, kt, vt, G, page, k, v, q=None, qname="float16", gate=None):
        n_kv, hd = k[0].shape[1:]
        self.lens, self.kt, self.vt, self.n_kv, self.nh, self.hd, self.page, self.qname = lens, kt, vt, n_kv, n_kv * G, hd, page, qname
        need = [ref.pages(p + n, page) for p, n in lens]
        self.n_pages, self.width = sum(need) + 1, max(need) + 1
        ids = np.split(rng.permutation(self.n_pages), np.cumsum(need))
        self.table = np.full((len(lens), self.width), -7, np.int32)
        self.k, self.v = (ref.Pool(t, self.n_pages, page, n_kv, hd, fill=0xff) for t in (kt, vt))   # NaN where nothing is written
        for i in range(len(lens)):
            self.table[i, :need[i]] = ids[i]
            self.k.write(ids[i], k[i])
            self.v.write(ids[i], v[i])
        self.start = np.concatenate([[0], np.cumsum([n for _, n in lens])])
        self.ntok = int(self.start[-1]) + 2
        t = torch()
        q = rng.standard_normal((self.ntok, self.nh, hd)) if q is None else q
        self.tq = t.from_numpy(np.asarray(q, np.float32)).to(getattr(t, qname)).cuda()
        self.gate, self.scale = gate, float(np.float32(hd ** -0.5))

    def output(self, rmi, split, **kw):
        self.run(rmi, split, q8=False, **kw)
        assert (self.y[self.start[-1]:] == 77.0).all()
        return self.y.double()

    def rows(self, i):
        s = slice(int(self.start[i]), int(self.start[i + 1]))
        return s, self.lens[i][0] + torch().arange(self.lens[i][1], device="cuda")


def marks_of(total, n_kv, hd, by):
    return np.repeat(exact.marks(total, hd, by).numpy()[:, None], n_kv, 1)


def count(got, pos, hd, by, one):
    """All weights of a row are equal (its keys are), so y times the positions seen is the number of marks at each dim times the value
    that a mark is held as.  A mark's share is off by the weights' rounding, y's own, and fp32 sums (a few hundred additions one after
    another at the sizes here, 2^-15): below half a mark for fewer than 490 marks a dim in fp16, 60 in bf16"""
    want = exact.marked(pos, hd, by).unsqueeze(1)
    n = got * (pos + 1).view(-1, 1, 1) / one
    assert bool((n.round() == want).all()), f"{int((n.round() != want).sum())} counts differ"
    assert bool(((n - want).abs() <= 0.5).all())


# past, new, heads of a KV head, head_dim, split
COUNTED = [(9000, 1, 4, 128, 128), (9000, 1, 16, 256, 1152), (39999, 1, 4, 128, 128), (119999, 1, 2, 256, 128), (119999, 1, 4, 256, 16384),
           (5003, 8, 4, 128, 128), (5003, 5, 4, 256, 640), (3001, 40, 4, 128, 128), (3001, 70, 4, 256, 512), (9000, 33, 4, 256, 9216)]


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("past,new,G,hd,split", COUNTED)
def test_every_position_counts_once(rmi, kt, vt, past, new, G, hd, split):
    """few rows, two blocks, tiles; joins of up to 1024 chunks; a short request beside the long one"""
    rng = np.random.default_rng(past + new)
    lens = [(past, new), (45, new)]
    one = kv_ref.held(marks_of(1, 1, hd, 1), vt).max()
    for by in (1, 32):
        k = [np.broadcast_to(rng.standard_normal((1, 1, hd)), (p + n, 1, hd)) for p, n in lens]
        b = Given(rng, lens, kt, vt, G, 256 if past > 10000 else 32, k, [marks_of(p + n, 1, hd, by) for p, n in lens])
        got = b.output(rmi, split, max_ctx=131072 if split == 128 and past > 40000 else None)
        for i in range(2):
            s, pos = b.rows(i)
            count(got[s], pos, hd, by, one)


def needles(rng, lens, nh):
    """for every token and head a position that the token sees: ends of pages and chunks, its own, any"""
    out = []
    for p, n in lens:
        for t in range(n):
            last = p + t
            edges = [x for e in (0, 15, 16, 31, 32, 63, 64, 127, 128, 255, 256, 1023, 1024, 4095, 4096) for x in (e, last - e) if 0 <= x <= last]
            edges += [x for c in range(128, last, 128) for x in (c - 1, c)]
            own = rng.choice(edges, nh)
            any_ = rng.integers(0, last + 1, nh)
            out.append(np.where(rng.random(nh) < 0.7, own, any_))
    return np.array(out)


@pytest.mark.parametrize("qname", ["float16", "bfloat16"])
@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("lens,G,hd,split", [([(9000, 1), (127, 1), (128, 1), (0, 1)], 16, 128, 128), ([(20001, 1)], 16, 256, 2048),
                                             ([(3000, 4)] * 6, 4, 256, 256), ([(4000, 8), (31, 8)], 4, 128, 128), ([(3000, 100), (0, 50)], 4, 128, 128),
                                             ([(2500, 200), (0, 90)], 4, 256, 1024)])
def test_every_key_is_found(rmi, qname, kt, vt, lens, G, hd, split):
    """q is four times one of the keys, whose elements are 1 or -1: its score, 4 sqrt(hd), is 45 or more against a deviation of 4, so
    that y is that position's V.  Rounded: the weight, y"""
    rng = np.random.default_rng(hd + split + G)
    n_kv = 2
    k = [rng.choice([-1.0, 1.0], (p + n, n_kv, hd)) for p, n in lens]
    v = [rng.standard_normal((p + n, n_kv, hd)) for p, n in lens]
    at = needles(rng, lens, n_kv * G)
    req = np.repeat(np.arange(len(lens)), [n for _, n in lens])
    kv = np.arange(n_kv * G) // G
    q = np.zeros((len(at) + 2, n_kv * G, hd))
    for r in range(len(at)):
        q[r] = 4 * k[req[r]][at[r], kv]
    b = Given(rng, lens, kt, vt, G, 16, k, v, q, qname)
    got = b.output(rmi, split)[:len(at)].cpu().numpy()
    held = [kv_ref.held(x, vt) for x in v]
    want = np.stack([held[req[r]][at[r], kv] for r in range(len(at))])
    # what the other keys weigh: each e^(score - 4 sqrt(hd)), the scores taken from the keys themselves
    keys = [kv_ref.held(x, kt) for x in k]
    for r in range(0, len(at), 7):
        for h in (0, n_kv * G - 1):
            s = keys[req[r]][:lens[req[r]][0] + r - b.start[req[r]] + 1, kv[h]] @ q[r, h] * b.scale
            s = s - s[at[r, h]]
            s[at[r, h]] = -np.inf
            assert np.exp(s).sum() < 2.0 ** -14
    tol = (2.0 ** -11 + ref.HALF_STEP[qname] + 2.0 ** -20) * np.abs(want) + 2.0 ** -14 * 8
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("qname,kt,vt", [("float16", F16, F16), ("bfloat16", I8, I8), ("float16", I8, I4), ("bfloat16", I4, I4)])
@pytest.mark.parametrize("lens,G,hd,split", [([(9000, 1), (8191, 1), (300, 1)], 4, 256, 128), ([(40000, 1)], 4, 128, 128), ([(9000, 6), (77, 8)], 4, 128, 384),
                                             ([(6000, 130), (129, 1)], 4, 256, 2048), ([(6000, 65)], 5, 128, 128), ([(8001, 20)], 3, 256, 8064)])
@pytest.mark.parametrize("rise", [0.0, 120.0, -120.0])
def test_long_contexts(rmi, qname, kt, vt, lens, G, hd, split, rise):
    """rise: the scores grow (or fall) by this much over the context, so that a row's maximum moves in most steps (or never again)"""
    t = torch()
    rng = np.random.default_rng(hd + split)
    n_kv = 2
    way = rng.choice([-1.0, 1.0], hd)
    k = [rng.standard_normal((p + n, n_kv, hd)) + way * (rise / (2 * hd ** 0.5) * np.arange(p + n) / (p + n))[:, None, None] for p, n in lens]
    v = [rng.standard_normal((p + n, n_kv, hd)) for p, n in lens]
    ntok = sum(n for _, n in lens) + 2
    q = rng.standard_normal((ntok, n_kv * G, hd)) + 2 * way * (rise != 0)   # q . way / sqrt(hd) is 2 sqrt(hd): rise in all
    gate = rng.standard_normal((ntok, n_kv * G, 2, hd)).astype(np.float32)
    b = Given(rng, lens, kt, vt, G, 128 if hd == 128 else 16, k, v, q, qname, gate)
    got = b.output(rmi, split)
    for i in range(len(lens)):
        s, pos = b.rows(i)
        kk, vv = (t.from_numpy(x).cuda() for x in b.held(i))
        want, bound = exact.attention(b.tq[s].double(), kk, vv, pos, b.scale, 2.0 ** -11, ref.HALF_STEP[qname],
                                      t.from_numpy(gate[s, :, 1].astype(np.float64)).cuda())
        assert exact.outside(got[s], want, bound) == 0, f"request {i}: off by {float((got[s] - want).abs().max()):.3g}, bound {float(bound.max()):.3g}"


# ---- whole prompts ---------------------------------------------------------------------------------------------------------
def prompt(rmi, q, k, v, lens, gate=None):
    """q [rows, heads, hd], k and v of one type"""
    t = torch()
    n, nh, hd = q.shape
    n_kv = k.shape[1]
    y = t.full_like(q, 77.0)
    rmi.gqa_prompt_attn(q, nh * hd, k, n_kv * hd, v, n_kv * hd, ints(np.concatenate([[0], np.cumsum(lens)])), gate, 2 * nh * hd, y, nh * hd, None, 0,
                        len(lens), n, max(lens), nh, n_kv, hd, float(np.float32(hd ** -0.5)))
    assert bool((y[sum(lens):] == 77.0).all())
    return y.double()


def normal(seed, *shape):
    t = torch()
    return t.randn(shape, generator=t.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=t.float32)


# the eight-wave form alone and ragged, four waves, 32 rows in four parts
PROMPTS = [([8001], 4, 4, 256), ([4090], 8, 4, 128), ([4200, 1, 2500, 0, 1300], 4, 4, 256), ([1100, 3, 1501, 0, 260], 4, 4, 256), ([1030, 1500], 2, 4, 128),
           ([1501], 1, 4, 256), ([900], 2, 3, 128)]


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens,n_kv,G,hd", PROMPTS)
def test_prompts_count_every_row_once(rmi, name, lens, n_kv, G, hd):
    t = torch()
    n, dtype = sum(lens) + 3, getattr(t, name)
    q = normal(1, n, n_kv * G, hd).to(dtype)
    k = normal(2, 1, n_kv, hd).to(dtype).expand(n, -1, -1).contiguous()
    for by in (1, 32):
        if name == "bfloat16" and -(-max(lens) // (by * hd)) * by > 60:
            continue   # more marks a dim than bf16 tells apart
        v = t.cat([exact.marks(m, hd, by) for m in lens] + [t.full((3, hd), 9.0, dtype=t.float64)]).to(dtype).cuda()
        got = prompt(rmi, q, k, v.unsqueeze(1).expand(-1, n_kv, -1).contiguous(), lens)
        at = 0
        for m in lens:
            for r in range(0, m, 1024):
                pos = t.arange(r, min(m, r + 1024), device="cuda")
                count(got[at + r:at + r + len(pos)], pos, hd, by, 1.0)
            at += m


@pytest.mark.parametrize("rise", [0.0, 120.0, -120.0])
@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens,n_kv,G,hd", PROMPTS)
def test_long_prompts(rmi, name, lens, n_kv, G, hd, rise):
    t = torch()
    n, dtype, step = sum(lens) + 3, getattr(t, name), ref.HALF_STEP[name]
    way = t.sign(normal(5, hd))
    up = t.cat([t.arange(m, device="cuda") / max(m, 1) for m in lens] + [t.zeros(3, device="cuda")])
    q = (normal(6, n, n_kv * G, hd) + 2 * way * (rise != 0)).to(dtype)
    k = (normal(7, n, n_kv, hd) + way * (rise / (2 * hd ** 0.5) * up).view(-1, 1, 1)).to(dtype)
    v = normal(8, n, n_kv, hd).to(dtype)
    gate = normal(9, n, n_kv * G, 2, hd)
    got = prompt(rmi, q, k, v, lens, gate)
    at = 0
    for m in lens:
        rows = sorted({r for e in (0, 1, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 1000, 1024) for r in (e, m - 1 - e) if 0 <= r < m} |
                      {m // 2, m // 3} & set(range(m)))
        for part in [rows[i:i + 16] for i in range(0, len(rows), 16)]:
            pos = t.tensor(part, device="cuda")
            want, bound = exact.attention(q[at + pos].double(), k[at:at + m].double(), v[at:at + m].double(), pos, float(np.float32(hd ** -0.5)), step, step,
                                          gate[at + pos, :, 1].double())
            off = got[at + pos] - want
            assert exact.outside(got[at + pos], want, bound) == 0, f"prompt of {m}: off by {float(off.abs().max()):.3g}, bound {float(bound.max()):.3g}"
        at += m
