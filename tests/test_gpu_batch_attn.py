"""Attention of a batch over pages and over packed prompts against a 64-bit restatement (tests/batch_ref.py)."""
import numpy as np
import pytest

from . import batch_ref as ref
from . import kv_ref
from .gpu_util import torch

pytestmark = pytest.mark.gpu
F16, I8, I4 = kv_ref.F16, kv_ref.I8, kv_ref.I4


@pytest.fixture(scope="module")
def rmi():
    torch()
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def rounded(x, name):
    """numpy values as the 16-bit type holds them, and the tensor"""
    t = torch().from_numpy(np.asarray(x, np.float32)).to(getattr(torch(), name)).cuda()
    return t.double().cpu().numpy(), t


def ints(x):
    return torch().tensor(np.asarray(x, np.int32), dtype=torch().int32, device="cuda")


class Batch:
    """lens: (past, new) of each request; pages in any order, unwritten bytes of any value"""

    def __init__(self, rng, lens, kt, vt, n_kv, G, hd, page, qname="float16", gate=True, spare=3, scale_q=1.0):
        self.lens, self.kt, self.vt, self.n_kv, self.nh, self.hd, self.page, self.qname = lens, kt, vt, n_kv, n_kv * G, hd, page, qname
        need = [ref.pages(p + n, page) for p, n in lens]
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages)
        self.width = max(need + [1]) + 1
        self.table = np.full((len(lens), self.width), -7, np.int32)
        self.k, self.v = (ref.Pool(t, self.n_pages, page, n_kv, hd, rng=rng) for t in (kt, vt))
        at = 0
        self.rows = []
        for i, (p, n) in enumerate(lens):
            self.table[i, :need[i]] = ids[at:at + need[i]]
            rows = [rng.standard_normal((p + n, n_kv, hd)) for _ in range(2)]
            self.rows.append(rows)
            self.k.write(ids[at:at + need[i]], rows[0])
            self.v.write(ids[at:at + need[i]], rows[1])
            at += need[i]
        self.start = np.concatenate([[0], np.cumsum([n for _, n in lens])])
        self.ntok = int(self.start[-1]) + 2   # two rows of padding
        self.q, self.tq = rounded(rng.standard_normal((self.ntok, self.nh, hd)) * scale_q, qname)
        self.gate = rng.standard_normal((self.ntok, self.nh, 2, hd)).astype(np.float32) if gate else None
        self.scale = float(np.float32(hd ** -0.5))
        self.known = {}

    def held(self, i):
        n = sum(self.lens[i])
        ids = self.table[i, :ref.pages(n, self.page)]
        return self.k.read(ids, n), self.v.read(ids, n)

    def run(self, rmi, split=None, stream=None, max_new=None, max_ctx=None, q8=True, table=None, kv_len=None, pools=None):
        t = torch()
        total = [p + n for p, n in self.lens]
        max_ctx = max_ctx or max(total + [1])
        max_new = max_new or max([n for _, n in self.lens] + [1])
        split = split or rmi.gqa_paged_split(max(1, sum(total)), max_ctx, len(total), self.ntok, max_new, self.nh, self.n_kv, self.hd)
        ws = t.full((rmi.gqa_paged_workspace_bytes(self.ntok, max_ctx, self.nh, self.hd, split),), 0xff, dtype=t.uint8, device="cuda")
        y = t.full((self.ntok, self.nh, self.hd), 77.0, dtype=self.tq.dtype, device="cuda")
        blocks = t.full((self.ntok, self.nh * self.hd // 32 * 36), 0xee, dtype=t.uint8, device="cuda") if q8 else None
        pk, pv = pools or (t.from_numpy(x.raw).cuda() for x in (self.k, self.v))
        gate = t.from_numpy(self.gate).cuda() if self.gate is not None else None
        args = (self.tq, self.kt, pk, self.vt, pv, ints(self.table if table is None else table), self.width, ints(self.start),
                ints(total if kv_len is None else kv_len), gate, 2 * self.nh * self.hd, y, self.nh * self.hd, blocks,
                self.nh * self.hd // 32 * 36, ws, len(total), self.ntok, max_new, max_ctx, self.nh, self.n_kv, self.hd, self.page,
                self.n_pages, split, self.scale)
        self.args, self.y, self.blocks = args, y, blocks
        rmi.gqa_paged_attn(*args)
        return y.double().cpu().numpy(), None if blocks is None else blocks.cpu().numpy()

    def expect(self, i):
        if i not in self.known:
            self.known[i] = self.formula(i)
        return self.known[i]

    def formula(self, i):
        s, n = self.start[i], self.lens[i][1]
        gate = None if self.gate is None else self.gate[s:s + n, :, 1].astype(np.float64)
        k, v = self.held(i)
        return ref.attention(self.q[s:s + n], k, v, self.lens[i][0], self.scale, gate, 2.0 ** -11, ref.HALF_STEP[self.qname])

    def check(self, y, blocks=None, orc=None, only=None):
        for i, (p, n) in enumerate(self.lens):
            if only is not None and i not in only:
                continue
            want, bound = self.expect(i)
            got = y[self.start[i]:self.start[i] + n]
            off = np.abs(got - want)
            assert not (~(off <= bound)).any(), f"request {i} (past {p}, new {n}): off by {np.nanmax(off):.3g}, bound {bound.max():.3g}"
        assert (y[self.start[-1]:] == 77.0).all(), "rows behind the last request"
        if blocks is not None:
            assert (blocks[self.start[-1]:] == 0xee).all()


def check_q8(y, blocks, out_step):
    """the blocks stand for what y was rounded from: |y| within a step of the block and y's own rounding"""
    b = blocks.reshape(-1, 36)
    d = b[:, :2].copy().view(np.float16).astype(np.float64)
    total = b[:, 2:4].copy().view(np.float16).astype(np.float64)[:, 0]
    codes = b[:, 4:].view(np.int8).astype(np.float64)
    y = y.reshape(-1, 32)
    # half a code step, d's rounding to fp16 over up to 127 codes, y's rounding, subnormals
    assert (np.abs(codes * d - y) <= 0.5 * d * (1 + 2.0 ** -9) + 127 * d * 2.0 ** -11 + out_step * np.abs(y) * (1 + out_step) + 2.0 ** -18).all()
    assert (np.abs(total - y.sum(1)) <= 2.0 ** -11 * np.abs(total) + (out_step + 2.0 ** -19) * np.abs(y).sum(1) + 2.0 ** -20).all()


TYPES = [(F16, F16), (I8, I8), (I4, I4), (I8, I4)]
MANY = [(0, 1), (63, 1), (64, 3), (700, 4), (15, 16), (0, 33), (31, 5), (128, 0), (127, 1), (300, 130), (32, 2), (1, 1)]


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("n_kv,G,hd,page", [(4, 4, 256, 64), (2, 8, 128, 16), (1, 5, 128, 256), (3, 3, 256, 16)])
def test_paged(rmi, kt, vt, n_kv, G, hd, page):
    rng = np.random.default_rng(7 * hd + page + 3 * kt + vt)
    b = Batch(rng, MANY, kt, vt, n_kv, G, hd, page, "bfloat16" if kt == I8 else "float16")
    for split in (128, 256, 1024):   # seven chunks and a join, four, one
        y, blocks = b.run(rmi, split)
        b.check(y, blocks)
        used = slice(0, b.start[-1])
        check_q8(y[used], blocks[used], ref.HALF_STEP[b.qname])


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("lens,G", [([(0, 5), (31, 8), (32, 7), (95, 6), (127, 5), (128, 8), (700, 8), (1100, 5), (64, 1), (15, 0), (200, 4)], 4),
                                    ([(p, 1) for p in (0, 15, 31, 63, 64, 300)] + [(9, 0)], 24), ([(40, 32), (0, 17), (5, 31), (3, 1)], 1),
                                    ([(40, 6), (0, 4), (511, 3)], 5)])
def test_paged_drafts(rmi, kt, vt, lens, G):
    """17 to 32 rows a request beside fewer"""
    rng = np.random.default_rng(G + 7 * kt + vt)
    for hd, page, name in ((256, 64, "float16"), (128, 16, "bfloat16")):
        b = Batch(rng, lens, kt, vt, 2, G, hd, page, name, gate=G == 4)
        for split in (128, 256, 1280):
            y, blocks = b.run(rmi, split)
            b.check(y, blocks)
            used = slice(0, b.start[-1])
            check_q8(y[used], blocks[used], ref.HALF_STEP[b.qname])


@pytest.mark.parametrize("page", [32, 128])
@pytest.mark.parametrize("new", [1, 2, 4, 5, 16, 17, 32, 33, 65])
def test_paged_lengths(rmi, new, page):
    rng = np.random.default_rng(new * page)
    for hd, G in ((128, 4), (256, 4)):
        b = Batch(rng, [(p, new) for p in (0, 1, 16, 31, 33, 95, 127, 128, 129, 1100)], F16, F16, 1, G, hd, page, gate=False)
        for split in (None, 128, 1280):
            b.check(b.run(rmi, split, q8=False)[0])


def test_paged_many_chunks(rmi):
    rng = np.random.default_rng(5)
    for new in (1, 20):
        b = Batch(rng, [(9000, new)], I8, I8, 2, 4, 128, 64)
        b.check(b.run(rmi, 128)[0])


@pytest.mark.parametrize("qname", ["float16", "bfloat16"])
def test_paged_large_and_small_q(rmi, qname):
    rng = np.random.default_rng(11)
    for s in (2.0 ** -12, 24.0):
        b = Batch(rng, [(90, 1), (200, 40)], F16, F16, 2, 4, 128, 16, qname, scale_q=s)
        b.check(b.run(rmi, 128)[0])


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("new", [4, 7, 40])
def test_unseen_rows_have_no_part(rmi, kt, vt, new):
    """K and V of a new token that are NaN or infinite: the tokens before it do not notice, the others are not finite"""
    rng = np.random.default_rng(new + kt)
    b = Batch(rng, [(70, new), (0, new)], kt, vt, 2, 4, 128, 16, gate=False)
    plain, _ = b.run(rmi, 128)
    at = new // 2
    for i in range(2):
        p = b.lens[i][0] + at
        for pool in (b.k, b.v):
            page = pool.raw[b.table[i, p // 16]]
            if pool.type == F16:
                row = page.view(np.uint16).reshape(16, 2, 128)[p % 16]
                row[:, 5:90:7], row[0, 6] = 0x7e00, 0x7c00
            else:
                scales = page[16 * 2 * (128 if pool.type == I8 else 64):].reshape(2, 16, 4)
                scales[:, p % 16] = 0xff
    y, _ = b.run(rmi, 128)
    for i in range(2):
        s = b.start[i]
        assert np.array_equal(y[s:s + at], plain[s:s + at])
        assert not np.isfinite(y[s + at:s + new, :, 5]).any()
        k, v = b.held(i)
        if vt == F16:   # K finite again: only the dims of V that are not finite are not, in the rows that see them
            for pool in (b.k,):
                pool.write(b.table[i, :ref.pages(sum(b.lens[i]), 16)], b.rows[i][0])
    if vt == F16:
        y, _ = b.run(rmi, 128)
        for i in range(2):
            s = b.start[i]
            dims = np.zeros(128, bool)
            dims[5:90:7] = True
            assert not np.isfinite(y[s + at:s + new][..., dims]).any()
            assert np.array_equal(y[s:s + at], plain[s:s + at])
            clean = y[s + at:s + new, 4:][..., ~dims]   # KV head 1 has no infinity
            assert np.array_equal(clean, plain[s + at:s + new, 4:][..., ~dims])
            assert np.isinf(y[s + at:s + new, :4, 6]).all()


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4)])
@pytest.mark.parametrize("new", [1, 3, 7, 40])
def test_pages_that_are_none(rmi, new, kt, vt):
    rng = np.random.default_rng(new)
    b = Batch(rng, [(100, new), (200, new), (90, new), (60, new)], kt, vt, 2, 4, 128, 32)
    table = b.table.copy()
    table[0, 2] = b.n_pages          # positions 64 ..
    table[1, 0] = -1
    table[3, :] = 2 ** 30
    for split in (128, 1024):
        y, _ = b.run(rmi, split, table=table)
        for i in (0, 1, 3):
            assert np.isnan(y[b.start[i]:b.start[i + 1]]).all()
        b.check(y, only=[2])
    if new == 40:   # tokens before such a page do not see it
        table = b.table.copy()
        table[3, 2] = -5             # positions 64 .. 95, tokens 4 and on
        y, _ = b.run(rmi, 128, table=table)
        s = b.start[3]
        want, bound = b.expect(3)
        assert (np.abs(y[s:s + 4] - want[:4]) <= bound[:4]).all() and np.isnan(y[s + 4:s + 40]).all()
    # a length past the table's row
    y, _ = b.run(rmi, 128, kv_len=[100 + new, 200 + new, 90 + new, 32 * b.width + 5], max_ctx=32 * b.width + 5)
    assert np.isnan(y[b.start[3]:b.start[4]][-1]).all()
    b.check(y, only=[0, 1, 2])


def test_rows_that_are_left_or_zero(rmi):
    rng = np.random.default_rng(3)
    b = Batch(rng, [(100, 1), (50, 20), (70, 2), (40, 30)], F16, F16, 2, 4, 128, 32)
    for split in (128, 1024):
        y, _ = b.run(rmi, split, max_new=20)   # 30 new ones: past the bound
        b.check(y, only=[0, 1, 2])
        assert (y[b.start[3]:] == 77.0).all()
        y, _ = b.run(rmi, split, max_ctx=71)   # 101 positions, and 72
        b.check(y, only=[1, 3])
        assert (y[:1] == 77.0).all() and (y[b.start[2]:b.start[3]] == 77.0).all()
        # a refused request (no length): its rows are zeros; a length below the new tokens: those before position 0 are
        y, blocks = b.run(rmi, split, kv_len=[0, 5, 72, -3])
        assert (y[:1] == 0).all() and (y[b.start[1]:b.start[1] + 15] == 0).all() and (y[b.start[3]:b.start[4]] == 0).all()
        assert np.isfinite(y[b.start[1] + 15:b.start[2]]).all() and (y[b.start[1] + 15:b.start[2]] != 0).any()
        assert (blocks[:1] == 0).all()
        b.check(y, only=[2])


def test_row_starts_that_are_not(rmi):
    """row starts beyond the call, negative or descending lead nowhere outside it"""
    rng = np.random.default_rng(4)
    b = Batch(rng, [(100, 1), (50, 20), (70, 2)], F16, F16, 2, 4, 128, 32)
    for start in ([0, 1, 10 ** 9, 10 ** 9], [-5, -9, 3, 2], [7, 3, 1, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5]):
        b.run(rmi, 128)
        args = list(b.args)
        args[7] = ints(np.array(start, np.int64).astype(np.int32))
        rmi.gqa_paged_attn(*args)
        torch().cuda.synchronize()


def test_same_bits_graph_and_stream(rmi):
    t = torch()
    rng = np.random.default_rng(9)
    for lens in ([(300, 1), (20, 1)], [(300, 1), (200, 50), (0, 7)]):
        b = Batch(rng, lens, I8, I4, 2, 4, 256, 16)
        first, _ = b.run(rmi, 128)
        again, _ = b.run(rmi, 128)
        assert np.array_equal(first, again)
        other = t.cuda.Stream()
        other.wait_stream(t.cuda.current_stream())
        b.y.zero_()
        t.cuda.synchronize()
        rmi.gqa_paged_attn(*b.args, stream=other)
        other.synchronize()
        assert np.array_equal(b.y.double().cpu().numpy()[:b.start[-1]], first[:b.start[-1]])
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            rmi.gqa_paged_attn(*b.args)
        lengths = b.args[8]
        for shorter in (0, 1, 0):   # the lengths are read when it runs
            lengths.copy_(ints([p + n - shorter for p, n in lens]))
            b.y.zero_()
            graph.replay()
            t.cuda.synchronize()
            got = b.y.double().cpu().numpy()
            b.y.zero_()
            rmi.gqa_paged_attn(*b.args)
            t.cuda.synchronize()
            assert np.array_equal(got, b.y.double().cpu().numpy())
            if not shorter:
                assert np.array_equal(got[:b.start[-1]], first[:b.start[-1]])


def test_pool_past_32_bits(rmi):
    t = torch()
    rng = np.random.default_rng(2)
    page, n_kv, hd = 256, 4, 256
    per = page * n_kv * hd * 2
    n_pages = (1 << 32) // per + 5
    for new in (1, 40):
        b = Batch(rng, [(300, new)], F16, F16, n_kv, 4, hd, page, gate=False)
        pools = [t.zeros(n_pages, per, dtype=t.uint8, device="cuda") for _ in range(2)]
        far = [n_pages - 1, n_pages - 3]
        for pool, src in zip(pools, (b.k, b.v)):
            for at, i in zip(far, b.table[0, :2]):
                pool[at].copy_(t.from_numpy(src.raw[i]))
        table = b.table.copy()
        table[0, :2] = far
        keep, b.n_pages = b.n_pages, n_pages
        y, _ = b.run(rmi, 1024, table=table, pools=pools, q8=False)
        b.n_pages = keep
        b.check(y)
        del pools


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I8)])
def test_more_requests_than_lanes(rmi, kt, vt):
    """200 requests of no, one and many tokens: each of the forms has some of several waves' worth"""
    rng = np.random.default_rng(21 + kt)
    new = rng.choice([0, 1, 1, 2, 4, 33, 70], 200, p=[0.1, 0.3, 0.2, 0.2, 0.1, 0.06, 0.04])
    lens = [(int(p), int(n)) for p, n in zip(rng.integers(0, 400, 200), new)]
    b = Batch(rng, lens, kt, vt, 1, 4, 128, 16)
    for split in (128, 512):
        b.check(*b.run(rmi, split))
    b.check(*b.run(rmi))


def test_most_requests(rmi):
    rng = np.random.default_rng(3)
    lens = [(int(p), int(n)) for p, n in zip(rng.integers(0, 40, 4096), rng.integers(0, 3, 4096))]
    b = Batch(rng, lens, F16, F16, 1, 1, 128, 16, gate=False)
    b.check(*b.run(rmi))
    b.check(*b.run(rmi, max_new=20))   # both forms are launched, one has none


@pytest.mark.parametrize("new", [1, 6, 40])
def test_bounds_far_above(rmi, new):
    """bounds of the longest context and of all the tokens: the chunks are many and long, the lengths are what they are"""
    rng = np.random.default_rng(new)
    b = Batch(rng, [(300, new), (0, new), (31, 1)], I8, I8, 1, 4, 128, 32)
    y, blocks = b.run(rmi, max_ctx=1 << 30, max_new=1 << 30)
    b.check(y, blocks)


@pytest.mark.parametrize("qname", ["float16", "bfloat16"])
@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4)])
@pytest.mark.parametrize("new", [1, 7, 40])
def test_q_that_is_not_finite(rmi, qname, kt, vt, new):
    """one head of one token: its row is NaN, the others do not notice"""
    rng = np.random.default_rng(new)
    b = Batch(rng, [(200, new), (50, new)], kt, vt, 2, 4, 128, 16, qname)
    plain, _ = b.run(rmi, 128, q8=False)
    at = b.start[1] - 1
    for bad in (float("nan"), float("inf"), float("-inf")):
        b.tq[at, 5, 77] = bad
        y, _ = b.run(rmi, 128, q8=False)
        assert np.isnan(y[at, 5]).all()
        y[at, 5] = plain[at, 5]
        assert np.array_equal(y, plain)


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I4, I4)])
def test_shared_pages(rmi, kt, vt):
    """requests that read the same pages: each as if it were alone"""
    t = torch()
    rng = np.random.default_rng(12)
    b = Batch(rng, [(250, 6)] * 3 + [(240, 1), (0, 40)], kt, vt, 2, 4, 128, 16)
    b.table[1] = b.table[2] = b.table[0]
    b.table[3, :16] = b.table[0, :16]
    for split in (128, 256):
        b.check(*b.run(rmi, split))


def test_two_calls_at_once(rmi):
    """on two streams, each with a workspace of its own: the bits of each alone"""
    t = torch()
    rng = np.random.default_rng(14)
    b = [Batch(rng, [(900, 1), (2000, 4), (60, 30)], kt, kt, 4, 4, 256, 64) for kt in (F16, I8)]
    first = [x.run(rmi, 128) for x in b]
    streams = [t.cuda.Stream() for _ in b]
    for x in b:
        x.y.zero_()
        x.blocks.zero_()
    t.cuda.synchronize()
    for _ in range(5):
        for x, s in zip(b, streams):
            rmi.gqa_paged_attn(*x.args, stream=s)
    t.cuda.synchronize()
    for x, (y, blocks) in zip(b, first):
        used = slice(0, x.start[-1])
        assert np.array_equal(x.y.double().cpu().numpy()[used], y[used]) and np.array_equal(x.blocks.cpu().numpy()[used], blocks[used])


# ---- whole prompts -------------------------------------------------------------------------------------------------------
def prompt_case(rmi, rng, lens, name, n_kv, G, hd, gate=True, pad=0, q8=True, max_len=None, heads=None):
    """rows of q, k and v side by side in one tensor (pad elements between them); heads: those of each KV head that are looked at"""
    t = torch()
    nh, n = n_kv * G, sum(lens)
    width = (nh + 2 * n_kv) * hd + pad
    rows, tr = rounded(rng.standard_normal((n + 3, width)), name)
    q, k, v = rows[:, :nh * hd], rows[:, nh * hd:(nh + n_kv) * hd], rows[:, (nh + n_kv) * hd:(nh + 2 * n_kv) * hd]
    start = np.concatenate([[0], np.cumsum(lens)])
    g = rng.standard_normal((n + 3, nh, 2, hd)).astype(np.float32) if gate else None
    y = t.full((n + 3, nh * hd + 4), 77.0, dtype=tr.dtype, device="cuda")
    blocks = t.full((n + 3, nh * hd // 32 * 36 + 4), 0xee, dtype=t.uint8, device="cuda") if q8 else None
    scale = float(np.float32(hd ** -0.5))
    args = (tr, width, tr[:, nh * hd:], width, tr[:, (nh + n_kv) * hd:], width, ints(start), t.from_numpy(g).cuda() if gate else None,
            2 * nh * hd, y, nh * hd + 4, blocks, nh * hd // 32 * 36 + 4, len(lens), n + 3, max_len or max(lens + [1]), nh, n_kv, hd, scale)
    rmi.gqa_prompt_attn(*args)
    got = y.double().cpu().numpy()
    for i, m in enumerate(lens):
        s = start[i]
        if max_len and m > max_len:
            assert (got[s:s + m] == 77.0).all()
            continue
        some = np.arange(nh).reshape(n_kv, G)[:, heads or slice(None)].reshape(-1)
        want, bound = ref.attention(q[s:s + m].reshape(m, nh, hd)[:, some], k[s:s + m].reshape(m, n_kv, hd), v[s:s + m].reshape(m, n_kv, hd), 0,
                                    scale, None if g is None else g[s:s + m, some, 1].astype(np.float64), ref.HALF_STEP[name], ref.HALF_STEP[name])
        off = np.abs(got[s:s + m, :nh * hd].reshape(m, nh, hd)[:, some] - want)
        assert not (~(off <= bound)).any(), f"prompt {i} of {m}: off by {np.nanmax(off):.3g}, bound {bound.max():.3g}"
    assert (got[n:] == 77.0).all() and (got[:, nh * hd:] == 77.0).all()
    if q8:
        raw = blocks.cpu().numpy()
        assert (raw[n:] == 0xee).all() and (raw[:, -4:] == 0xee).all()
        if not max_len:
            check_q8(got[:n, :nh * hd], np.ascontiguousarray(raw[:n, :-4]), ref.HALF_STEP[name])
    return args, y


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("n_kv,G,hd", [(4, 4, 256), (2, 8, 128), (1, 5, 128), (3, 3, 256), (1, 1, 128)])
def test_prompts(rmi, name, n_kv, G, hd):
    rng = np.random.default_rng(hd + G)
    prompt_case(rmi, rng, [1, 0, 33, 2, 31, 32, 150, 64, 0], name, n_kv, G, hd)
    prompt_case(rmi, rng, [300], name, n_kv, G, hd, gate=False, pad=8, q8=False)


def test_prompts_many(rmi):
    rng = np.random.default_rng(8)
    prompt_case(rmi, rng, [int(x) for x in rng.integers(0, 9, 200)] + [70, 0, 3], "float16", 1, 4, 128)
    prompt_case(rmi, rng, [10, 90, 20, 91], "float16", 1, 4, 128, max_len=90)


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd", [128, 256])
def test_prompt_forms(rmi, name, hd):
    """the workgroups of eight waves, with heads enough for many of them, and those of four over prompts of several tiles"""
    rng = np.random.default_rng(hd)
    prompt_case(rmi, rng, [257, 0, 5], name, 8, 64, hd, gate=hd == 128, heads=[0, 63])
    prompt_case(rmi, rng, [150, 149, 151, 9, 180, 150, 150], name, 4, 4, hd, heads=[1])


@pytest.mark.parametrize("G", [4, 8])
@pytest.mark.parametrize("lens", [[70], [160, 3]])
def test_prompt_rows_far_apart(rmi, lens, G):
    """rows as far apart as may be, the last steps cut at the call's end"""
    t = torch()
    rng = np.random.default_rng(5)
    n, hd, stride = sum(lens), 128, 1 << 25
    far = t.empty(n, stride, dtype=t.float16, device="cuda")
    q, k, v = (rng.standard_normal((n, h, hd)).astype(np.float16) for h in (G, 1, 1))
    far[:, :hd] = t.from_numpy(k[:, 0]).cuda()
    far[:, hd:2 * hd] = t.from_numpy(v[:, 0]).cuda()
    y = t.empty(n, G, hd, dtype=t.float16, device="cuda")
    start, scale = np.concatenate([[0], np.cumsum(lens)]), float(np.float32(hd ** -0.5))
    rmi.gqa_prompt_attn(t.from_numpy(q).cuda(), G * hd, far, stride, far[:, hd:], stride, ints(start), None, 0, y, G * hd, None, 0, len(lens), n,
                        max(lens), G, 1, hd, scale)
    got = y.double().cpu().numpy()
    for s, m in zip(start, lens):
        want, bound = ref.attention(*(x[s:s + m].astype(np.float64) for x in (q, k, v)), 0, scale, None, 2.0 ** -11, 2.0 ** -11)
        assert (np.abs(got[s:s + m] - want) <= bound).all()


def test_prompt_large_values(rmi):
    """bf16 values near the type's largest: the sums on the way stay inside fp32 (a weight is at most 2^7, 100 of them)"""
    t = torch()
    rng = np.random.default_rng(17)
    for lens in ([100], [30] * 8):
        args, y = prompt_case(rmi, rng, lens, "bfloat16", 1, 8, 128, gate=False, q8=False)
        plain = y.double().cpu().numpy()
        rows = args[0]
        rows[:, 9 * 128:] *= 2.0 ** 110   # of the order of 2^112, times 2^14 for all the weights
        rmi.gqa_prompt_attn(*args)
        n = sum(lens)
        got = y.double().cpu().numpy()[:n, :1024]
        assert np.array_equal(got, plain[:n, :1024] * 2.0 ** 110)


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens,n_kv,G", [([100, 40], 1, 8), ([20] * 30, 2, 4), ([257, 9], 8, 64)])
def test_prompt_q_that_is_not_finite(rmi, name, lens, n_kv, G):
    rng = np.random.default_rng(G)
    args, y = prompt_case(rmi, rng, lens, name, n_kv, G, 128, gate=False, q8=False, heads=[0])
    plain = y.double().cpu().numpy()
    at, h = lens[0] - 1, n_kv * G - 2
    for bad in (float("nan"), float("inf"), float("-inf")):
        args[0][at, 128 * h + 5] = bad
        rmi.gqa_prompt_attn(*args)
        got = y.double().cpu().numpy()
        mine = slice(128 * h, 128 * (h + 1))
        assert np.isnan(got[at, mine]).all()
        got[at, mine] = plain[at, mine]
        assert np.array_equal(got, plain)


@pytest.mark.parametrize("lens,n_kv,G", [([100, 40, 3], 1, 8), ([20] * 30, 2, 4), ([257, 9, 2], 8, 64)])
def test_prompt_row_starts_that_are_not(rmi, lens, n_kv, G):
    """row starts beyond the call, negative or descending lead nowhere outside it"""
    rng = np.random.default_rng(4)
    args, y = prompt_case(rmi, rng, lens, "bfloat16", n_kv, G, 128, gate=False, q8=False, heads=[0])
    for start in ([0, 1, 10 ** 9, 10 ** 9], [-5, -9, 3, 2], [7, 3, 1, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5], [0, 200, 0, 200]):
        args[6][:4] = ints(np.array(start, np.int64).astype(np.int32))
        rmi.gqa_prompt_attn(*args)
        torch().cuda.synchronize()


@pytest.mark.parametrize("lens,n_kv,G", [([100, 40], 1, 8), ([20] * 30, 2, 4), ([257, 9], 8, 64)])
def test_prompt_graph_and_stream(rmi, lens, n_kv, G):
    """a captured call reads the row starts when it runs; on another stream the same bits"""
    t = torch()
    rng = np.random.default_rng(len(lens))
    args, y = prompt_case(rmi, rng, lens, "float16", n_kv, G, 128, heads=[1])
    first, start, blocks = y.clone(), args[6], args[11]
    other = t.cuda.Stream()
    other.wait_stream(t.cuda.current_stream())
    y.fill_(77.0)
    t.cuda.synchronize()
    rmi.gqa_prompt_attn(*args, stream=other)
    other.synchronize()
    assert t.equal(y, first)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        rmi.gqa_prompt_attn(*args)
    keep = start.clone()
    for cut in (0, 7, 3, 0):   # the first prompt's last rows become the second's first
        start.copy_(keep)
        start[1:-1] -= cut
        got = []
        for run in (graph.replay, lambda: rmi.gqa_prompt_attn(*args)):
            y.fill_(77.0)
            blocks.fill_(0xee)
            t.cuda.synchronize()
            run()
            t.cuda.synchronize()
            got.append((y.clone(), blocks.clone()))
        assert t.equal(got[0][0], got[1][0]) and t.equal(got[0][1], got[1][1])
        assert t.equal(got[0][0], first) == (cut == 0)


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("lens,n_kv,G", [([40, 100, 9], 1, 4), ([40, 100, 9], 1, 3), ([40, 257, 9], 8, 64), ([40, 100, 9] + [90] * 18, 1, 4)])
def test_prompt_unseen_rows(rmi, name, hd, lens, n_kv, G):
    """a row whose k and v are not finite: no part in the rows before it, nor in other prompts"""
    rng = np.random.default_rng(6)
    args, y = prompt_case(rmi, rng, lens, name, n_kv, G, hd, gate=False, q8=False, heads=[0])
    plain = y.double().cpu().numpy()
    row, nh, end = args[0], n_kv * G, 40 + lens[1]
    k, v = row[:, nh * hd:(nh + 1) * hd], row[:, (nh + n_kv) * hd:(nh + n_kv + 1) * hd]   # KV head 0
    keep = k[70].clone(), v[70].clone()
    v[70, 3:60:5] = float("nan")
    v[70, 64] = float("inf")
    for k_too in (False, True):
        if k_too:
            k[70] = float("nan")
        rmi.gqa_prompt_attn(*args)
        got = y.double().cpu().numpy()
        before = np.r_[0:70, end:len(got)]
        assert np.array_equal(got[before], plain[before])
        assert np.array_equal(got[:, G * hd:], plain[:, G * hd:])
        after = got[70:end, :G * hd].reshape(end - 70, G, hd)
        odd = np.zeros(hd, bool)
        odd[3:60:5] = odd[64] = True
        assert not np.isfinite(after[..., odd]).any()
        if k_too:
            assert np.isnan(after).all()
        else:
            assert np.array_equal(after[..., ~odd], plain[70:end, :G * hd].reshape(end - 70, G, hd)[..., ~odd]) and np.isinf(after[..., 64]).all()
    k[70], v[70] = keep
    rmi.gqa_prompt_attn(*args)
    assert np.array_equal(y.double().cpu().numpy(), plain)


def test_prompt_equals_pages(rmi):
    """a prompt over its packed rows and over an fp16 page pool whose slots are in order: the same rows.  The forms add a row's weights
    in different orders, so each is held to the formula by its bound, and with it to the other"""
    t = torch()
    rng = np.random.default_rng(1)
    n, n_kv, G, hd = 200, 2, 4, 256
    nh = n_kv * G
    q, k, v = (t.from_numpy(rng.standard_normal((256, h, hd)).astype(np.float16)).cuda() for h in (nh, n_kv, n_kv))
    y = [t.empty(n, nh, hd, dtype=t.float16, device="cuda") for _ in range(2)]
    start, scale = ints([0, n]), hd ** -0.5
    rmi.gqa_prompt_attn(q, nh * hd, k, n_kv * hd, v, n_kv * hd, start, None, 0, y[0], nh * hd, None, 0, 1, n, n, nh, n_kv, hd, scale)
    rmi.gqa_paged_attn(q, rmi.KV_F16, k, rmi.KV_F16, v, ints([0, 1, 2, 3]), 4, start, ints([n]), None, 0, y[1], nh * hd, None, 0, None, 1, n,
                       n, n, nh, n_kv, hd, 64, 4, 256, scale)
    want, bound = ref.attention(*(x[:n].double().cpu().numpy() for x in (q, k, v)), 0, float(np.float32(scale)), None, 2.0 ** -11, 2.0 ** -11)
    for got in y:
        assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
