"""Page plans, trims, rows of slots and the prep into pages against plain restatements (tests/batch_ref.py), and rounds of a batch."""
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


def ints(x):
    return torch().tensor(np.asarray(x, np.int64).astype(np.int32), dtype=torch().int32, device="cuda")


def run_plan(rmi, past, count, page, n_pages, free, n_free, table, max_tok):
    n, width = table.shape
    tt = ints(table)
    out = [torch().full((k,), -99, dtype=torch().int32, device="cuda") for k in (n + 1, n, max_tok, max_tok, 1, n)]
    args = (ints(past), ints(count), n, page, n_pages, ints(free), ints([n_free]), tt, width, max_tok, *out)
    rmi.page_plan(*args)
    return [x.cpu().tolist() for x in out] + [tt.cpu().numpy()], args


def compare_plan(got, want, past, count):
    row_start, kv_len, slot, pos, n_left, status, table = want
    assert got[0] == row_start and got[1] == kv_len and got[2] == slot and got[4] == [n_left] and got[5] == status
    good = [i for i, s in enumerate(status) if s != 1]   # positions of a request with bad lengths are anything
    for i in good:
        assert got[3][row_start[i]:row_start[i + 1]] == pos[row_start[i]:row_start[i + 1]]
    assert got[3][row_start[-1]:] == pos[row_start[-1]:]
    assert np.array_equal(got[6], table)


def batch(rng, n, page, ctx, new, spare):
    past = rng.integers(0, ctx + 1, n)
    count = rng.integers(0, new + 1, n)
    past[rng.random(n) < 0.2] = 0
    width = ref.pages(ctx + new, page)
    held = [ref.pages(p, page) for p in past]
    need = sum(ref.pages(p + c, page) - h for p, c, h in zip(past, count, held))
    n_free = int(need * spare)
    n_pages = sum(held) + n_free + 1
    ids = rng.permutation(n_pages)
    table = np.full((n, width), -1, np.int32)
    at = n_free
    for i in range(n):
        table[i, :held[i]] = ids[at:at + held[i]]
        at += held[i]
    free = np.full(n_pages, -3, np.int32)
    free[:n_free] = ids[:n_free]
    return past, count, n_pages, free, n_free, table


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("n,ctx,new,spare", [(1, 40, 1, 1), (1, 0, 5000, 1), (3, 100, 60, 1.0), (64, 300, 1, 1.2), (65, 300, 16, 0.6),
                                             (257, 1000, 40, 0.9), (1000, 90, 33, 1), (4096, 50, 3, 0.5)])
def test_plan(rmi, n, ctx, new, spare, page):
    rng = np.random.default_rng(n + page)
    past, count, n_pages, free, n_free, table = batch(rng, n, page, ctx, new, spare)
    for max_tok in (int(count.sum()) + 7, max(1, int(count.sum()))):
        got, args = run_plan(rmi, past, count, page, n_pages, free, n_free, table, max_tok)
        compare_plan(got, ref.plan(past, count, page, n_pages, free, n_free, table, max_tok), past, count)
        rmi.page_plan(*args)   # the table that it filled gives the same plan
        assert [x.cpu().tolist() for x in args[10:]] == got[:6] and np.array_equal(args[7].cpu().numpy(), got[6])


def test_plan_lengths_that_are_not(rmi):
    rng = np.random.default_rng(1)
    past, count, n_pages, free, n_free, table = batch(rng, 40, 16, 200, 20, 2.0)
    past, count = past.astype(np.int64), count.astype(np.int64)
    past[3], past[5], count[7], count[9], past[11] = -1, 2 ** 31 - 1, -4, 2 ** 31 - 1, table.shape[1] * 16 + 1
    count[5] = 2 ** 31 - 1
    got, _ = run_plan(rmi, past, count, 16, n_pages, free, n_free, table, 300)
    compare_plan(got, ref.plan(past, count, 16, n_pages, free, n_free, table, 300), past, count)
    for n in (-5, 10 ** 9):   # a count of free pages is brought into range
        got, _ = run_plan(rmi, past, count, 16, n_pages, free, n, table, 300)
        compare_plan(got, ref.plan(past, count, 16, n_pages, free, min(max(n, 0), n_pages), table, 300), past, count)


@pytest.mark.parametrize("n", [1, 3, 64, 300, 4096])
@pytest.mark.parametrize("page", [16, 128])
def test_trim(rmi, n, page):
    rng = np.random.default_rng(n * page)
    length, _, n_pages, free, n_free, table = batch(rng, n, page, 700, 0, 1)
    keep = np.minimum(length, rng.integers(0, 701, n))
    keep[rng.random(n) < 0.3] = 0
    keep[0] = length[0]
    if n > 3:
        keep[1], keep[2] = -1, length[2] + 1
    for room in (n_pages, max(1, n_pages // 3)):
        f = ints(free)
        out = ints([-1])
        rmi.page_trim(ints(length), ints(keep), n, page, room, ints(table), table.shape[1], ints([min(n_free, room)]), f[:room], out)
        at, want = ref.trim(length, keep, page, room, table, min(n_free, room), free[:room].tolist())
        assert out.item() == at and f[:room].cpu().tolist() == want
        assert f[room:].cpu().tolist() == free[room:].tolist()


def test_trim_long_lengths(rmi):
    """lengths past the table's row end with it"""
    f, out, table = ints([-1] * 9), ints([-1]), np.arange(8).reshape(2, 4)
    rmi.page_trim(ints([2 ** 31 - 1, 64]), ints([17, 0]), 2, 16, 9, ints(table), 4, ints([0]), f, out)
    assert out.item() == 6 and f.cpu().tolist() == [2, 3, 4, 5, 6, 7, -1, -1, -1]


# ---- prep and rows of slots ------------------------------------------------------------------------------------------------
EPS, BASE = 1e-6, 1e7
LONG = {"factor": 4.0, "orig_ctx": 8192.0, "beta_fast": 32.0, "beta_slow": 1.0}


def prep(rmi, rng, kt, vt, n_kv, G, hd, n_rot, neighbours, name, n, page, norms=(True, True), stride_pad=0, far=False, scale=1.0, rope=None):
    t = torch()
    nh = n_kv * G
    width = 2 * nh * hd + 2 * n_kv * hd
    q3 = (rng.standard_normal((n, width + stride_pad)) * scale).astype(np.float32)
    n_pages = ref.pages(n, page) + 2
    slot = rng.permutation(n_pages * page)[:n].astype(np.int64)
    if n > 2:
        slot[1], slot[2] = -1, n_pages * page   # rows that go nowhere
    pos = rng.integers(0, 2 ** 20 if far else 3000, n)
    w = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if use else None for use in norms]
    pools = [t.zeros(n_pages, ref.Pool(x, 1, page, n_kv, hd, fill=0).raw.shape[1], dtype=t.uint8, device="cuda") for x in (kt, vt)]
    q = t.full((n, nh, hd), 77.0, dtype=getattr(t, name), device="cuda")
    dev = [None if x is None else t.from_numpy(x).cuda() for x in w]
    args = (t.from_numpy(q3).cuda(), width + stride_pad, dev[0], dev[1], kt, pools[0], vt, pools[1], ints(slot), ints(pos), q, nh, n_kv, hd, n_rot,
            rmi.ROPE_NEIGHBOURS if neighbours else rmi.ROPE_HALF, BASE, EPS, n, page, n_pages)
    rmi.attn_prep_paged(*args, **(rope or {}))
    rope = dict(rope or {})
    kw = {"factor": rope.get("factor", 1.0), "orig": rope.get("orig_ctx", 0.0), "ext": rope.get("ext_factor", 1.0)}
    used = (slot >= 0) & (slot < n_pages * page)
    heads = q3[:, :2 * nh * hd].reshape(n, nh, 2, hd)[:, :, 0]
    rows = q3[:, 2 * nh * hd:width].reshape(n, 2, n_kv, hd)
    want_q = ref.rotated(heads, w[0], pos, n_rot, neighbours, EPS, BASE, **kw)
    want_k = ref.rotated(rows[:, 0], w[1], pos, n_rot, neighbours, EPS, BASE, **kw)
    return args, q, pools, slot, used, want_q, want_k, rows[:, 1].astype(np.float64), n_pages


def near(got, want, row_max, step, what):
    """fp32 norm and rotation: hd / 2 + 8 roundings of 2^-24 in the norm's sum and its root, four more, relative to a row's largest
    (a pair mixes two dims); the result rounded once (step)"""
    tol = 2.0 ** -24 * 160 * row_max + step * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -24
    assert (np.abs(got - want) <= tol).all(), what


def check_prep(rmi, out, kt, vt, n_kv, hd, page, name):
    t = torch()
    args, q, pools, slot, used, want_q, want_k, want_v, n_pages = out
    got = q.double().cpu().numpy()
    near(got[used], want_q[used], np.abs(want_q[used]).max(-1, keepdims=True), ref.HALF_STEP[name], "q")
    assert (got[~used] == 77.0).all()
    n = len(slot)
    for type_, pool, want, what in ((kt, pools[0], want_k, "k"), (vt, pools[1], want_v, "v")):
        held = kv_ref.held(want.astype(np.float32), type_)
        raw = pool.cpu().numpy()
        values = np.stack([kv_ref.decode(x, type_, page, n_kv, hd) for x in raw]).reshape(-1, n_kv, hd)
        rows = np.zeros_like(want)
        rows[used] = values[slot[used]]
        # K in fp64: it and the fp64 here differ by some 2^-45, so a code or a rounding differs where a value lies that near a
        # border (one in 10^9): none of these rows, which are fixed
        assert np.array_equal(rows[used], held[used]), what
        untouched = np.ones(len(values), bool)
        untouched[slot[used]] = False
        empty = kv_ref.decode(np.zeros_like(raw[0]), type_, page, n_kv, hd)[0, 0, 0]
        assert (values[untouched] == empty).all()
        for dtype, stride in ((t.float32, n_kv * hd), (t.float16, n_kv * hd + 2), (t.float16, n_kv * hd + 8)):
            back = t.full((n, stride), 55.0, dtype=dtype, device="cuda")
            rmi.kv_page_read(type_, pool, args[8], back, stride, n, n_kv, hd, page, n_pages)
            b = back.double().cpu().numpy()
            assert np.array_equal(b[:, :n_kv * hd].reshape(n, n_kv, hd)[used], rows[used])
            assert (b[:, :n_kv * hd][~used] == 0).all() and (b[:, n_kv * hd:] == 55.0).all()


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I8), (I8, I4), (I4, I4), (F16, I8), (I4, F16)])
@pytest.mark.parametrize("n_kv,G,hd,n_rot,neighbours,name", [(4, 4, 256, 64, False, "float16"), (2, 4, 128, 128, True, "bfloat16"),
                                                             (1, 5, 128, 30, False, "float16"), (3, 3, 256, 256, True, "float16"),
                                                             (1, 1, 256, 6, True, "bfloat16"), (2, 8, 128, 0, False, "float16"),
                                                             (1, 2, 256, 254, False, "bfloat16")])
def test_prep(rmi, kt, vt, n_kv, G, hd, n_rot, neighbours, name):
    rng = np.random.default_rng(hd + n_rot + 10 * kt + vt)
    for n, page in ((1, 16), (45, 32)):
        out = prep(rmi, rng, kt, vt, n_kv, G, hd, n_rot, neighbours, name, n, page, stride_pad=3 if n > 1 else 0)
        check_prep(rmi, out, kt, vt, n_kv, hd, page, name)


@pytest.mark.parametrize("rope", [LONG, {**LONG, "factor": 8.0, "ext_factor": 0.0}, {"factor": 0.5}])
@pytest.mark.parametrize("neighbours", [False, True])
def test_prep_scaled_and_far(rmi, rope, neighbours):
    rng = np.random.default_rng(5)
    out = prep(rmi, rng, F16, I8, 2, 4, 256, 64, neighbours, "float16", 300, 64, far=True, rope=rope)
    args, q, pools, slot, used, want_q, want_k, want_v, n_pages = out
    got = q.double().cpu().numpy()
    near(got[used], want_q[used], np.abs(want_q[used]).max(-1, keepdims=True), 2.0 ** -11, "q")
    values = np.stack([kv_ref.decode(x, F16, 64, 2, 256) for x in pools[0].cpu().numpy()]).reshape(-1, 2, 256)
    near(values[slot[used]], want_k[used], np.abs(want_k[used]).max(-1, keepdims=True) * 2.0 ** -10, 2.0 ** -11, "k")


@pytest.mark.parametrize("norms", [(False, False), (True, False), (False, True)])
def test_prep_without_norms(rmi, norms):
    rng = np.random.default_rng(9)
    out = prep(rmi, rng, I8, I8, 2, 4, 128, 64, False, "bfloat16", 20, 16, norms=norms, scale=3.0)
    check_prep(rmi, out, I8, I8, 2, 128, 16, "bfloat16")


def test_prep_many_tokens_and_large_pools(rmi):
    """a thousand tokens (several rows a wave), slots past 2^32 bytes"""
    t = torch()
    rng = np.random.default_rng(4)
    out = prep(rmi, rng, I8, I4, 4, 4, 256, 64, False, "float16", 999, 64)
    check_prep(rmi, out, I8, I4, 4, 256, 64, "float16")
    args, q = list(out[0]), out[1]
    per = 256 * 4 * 512
    n_pages = (1 << 32) // per + 3
    big = [t.zeros(n_pages, per, dtype=t.uint8, device="cuda") for _ in range(2)]
    slot = ints((n_pages - 1) * 256 + np.array([5, 255, 0]))
    args[0], args[4:10] = args[0][:3].contiguous(), [F16, big[0], F16, big[1], slot, args[9][:3].contiguous()]
    args[18:] = [3, 256, n_pages]
    args[10] = t.empty(3, 16, 256, dtype=t.float16, device="cuda")
    rmi.attn_prep_paged(*args)
    for pool, want in ((big[0], out[6]), (big[1], out[7])):
        got = pool[-1].view(t.float16).view(256, 4, 256)[[5, 255, 0]].double().cpu().numpy()
        assert np.array_equal(got, kv_ref.held(want[:3].astype(np.float32), F16))
        back = t.empty(3, 1024, dtype=t.float32, device="cuda")
        rmi.kv_page_read(F16, pool, slot, back, 1024, 3, 4, 256, 256, n_pages)
        assert np.array_equal(back.double().cpu().numpy().reshape(3, 4, 256), got)
        assert not pool[:-1].any()


def test_prep_graph_and_stream(rmi):
    t = torch()
    rng = np.random.default_rng(12)
    out = prep(rmi, rng, I8, I8, 2, 4, 256, 64, False, "float16", 40, 32)
    args, q, pools = out[0], out[1], out[2]
    first = q.clone(), pools[0].clone(), pools[1].clone()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        rmi.attn_prep_paged(*args)
    for _ in range(3):
        q.fill_(77.0)
        pools[0].zero_(), pools[1].zero_()
        graph.replay()
        t.cuda.synchronize()
        assert t.equal(q, first[0]) and t.equal(pools[0], first[1]) and t.equal(pools[1], first[2])
    other = t.cuda.Stream()
    q.fill_(77.0)
    t.cuda.synchronize()
    rmi.attn_prep_paged(*args, stream=other)
    other.synchronize()
    assert t.equal(q, first[0])


# ---- rounds ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4)])
@pytest.mark.parametrize("captured", [False, True])
def test_rounds(rmi, kt, vt, captured):
    """Requests that arrive, decode, draft, lose drafts and end, in one pool: plan, prep, attention, trim, against each request's
    own history; the first prompts by both calls"""
    t = torch()
    rng = np.random.default_rng(21)
    n, page, n_pages, n_kv, G, hd, n_rot, width, most = 5, 16, 60, 2, 4, 128, 64, 20, 300
    nh = n_kv * G
    w3 = 2 * nh * hd + 2 * n_kv * hd
    wq, wk = (t.from_numpy((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)).cuda() for _ in range(2))
    bytes_of = [ref.Pool(x, 1, page, n_kv, hd, fill=0).raw.shape[1] for x in (kt, vt)]
    pools = [t.from_numpy(rng.integers(0, 256, (n_pages, b), dtype=np.uint8)).cuda() for b in bytes_of]
    table, free = ints(np.full((n, width), -1)), ints(rng.permutation(n_pages))
    n_free, n_left = ints([n_pages]), ints([0])
    past, count, keep = ints([0] * n), ints([0] * n), ints([0] * n)
    row_start, kv_len, status = ints([0] * (n + 1)), ints([0] * n), ints([0] * n)
    slot, pos = ints([0] * most), ints([0] * most)
    q3 = t.zeros(most, w3, device="cuda")
    q, y = (t.zeros(most, nh, hd, dtype=t.float16, device="cuda") for _ in range(2))
    max_ctx, scale = width * page, float(np.float32(hd ** -0.5))
    split = 128
    ws = t.empty(rmi.gqa_paged_workspace_bytes(most, max_ctx, nh, hd, split), dtype=t.uint8, device="cuda")

    def round_():
        rmi.page_plan(past, count, n, page, n_pages, free, n_free, table, width, most, row_start, kv_len, slot, pos, n_left, status)
        rmi.attn_prep_paged(q3, w3, wq, wk, kt, pools[0], vt, pools[1], slot, pos, q, nh, n_kv, hd, n_rot, rmi.ROPE_HALF, BASE, EPS, most, page,
                            n_pages)
        rmi.gqa_paged_attn(q, kt, pools[0], vt, pools[1], table, width, row_start, kv_len, q3, w3, y, nh * hd, None, 0, ws, n, most, most,
                           max_ctx, nh, n_kv, hd, page, n_pages, split, scale)

    def end():
        rmi.page_trim(kv_len, keep, n, page, n_pages, table, width, n_left, free, n_free)

    graphs = None
    if captured:
        graphs = [t.cuda.CUDAGraph() for _ in range(2)]
        for g, f in zip(graphs, (round_, end)):
            with t.cuda.graph(g):
                f()
    lengths = [0] * n
    hist = [(np.zeros((0, n_kv, hd)), np.zeros((0, n_kv, hd))) for _ in range(n)]
    for counts, kept in (([40, 7, 0, 100, 1], None), ([1, 1, 33, 1, 1], [1, 1, 33, 1, 1]), ([1, 5, 1, 0, 5], [1, 2, 1, 0, 5]),
                         ([1, 4, 1, 1, 1], [1, 0, 1, -1, 1]), ([5, 1, 5, 70, 16], [3, 1, 5, 70, 16])):
        kept = kept or counts
        past.copy_(ints(lengths)), count.copy_(ints(counts))
        x = rng.standard_normal((most, w3)).astype(np.float32)
        q3.copy_(t.from_numpy(x))
        y.fill_(77.0)
        t.cuda.synchronize()
        graphs[0].replay() if captured else round_()
        t.cuda.synchronize()
        assert status.cpu().tolist() == [0] * n
        got, start, positions = y.double().cpu().numpy(), np.concatenate([[0], np.cumsum(counts)]), pos.cpu().numpy()
        assert row_start.cpu().tolist() == start.tolist()
        live = [p for i in range(n) for p in table[i, :ref.pages(lengths[i] + counts[i], page)].cpu().tolist()]
        assert len(set(live)) == len(live) and all(0 <= p < n_pages for p in live)
        assert n_left.item() == n_pages - len(live) and not set(live) & set(free[:n_left.item()].cpu().tolist())
        held_q = q.double().cpu().numpy()
        for i, c in enumerate(counts):
            rows = slice(start[i], start[i + 1])
            if c == 0:
                continue
            k = ref.rotated(x[rows, 2 * nh * hd:].reshape(c, 2, n_kv, hd)[:, 0], wk.double().cpu().numpy(), positions[rows], n_rot, False, EPS, BASE)
            v = x[rows, 2 * nh * hd:].reshape(c, 2, n_kv, hd)[:, 1]
            all_k = np.concatenate([hist[i][0], kv_ref.held(k.astype(np.float32), kt)])
            all_v = np.concatenate([hist[i][1], kv_ref.held(v, vt)])
            gate = x[rows, :2 * nh * hd].reshape(c, nh, 2, hd)[:, :, 1].astype(np.float64)
            want, bound = ref.attention(held_q[rows], all_k, all_v, lengths[i], scale, gate, 2.0 ** -11, 2.0 ** -11)
            assert (np.abs(got[rows] - want) <= bound).all(), f"request {i}: {np.abs(got[rows] - want).max()}"
            stay = lengths[i] + kept[i] if kept[i] >= 0 else 0
            hist[i] = all_k[:stay], all_v[:stay]
        assert (got[start[-1]:] == 77.0).all()
        lengths = [a + k if k >= 0 else 0 for a, k in zip(lengths, kept)]
        keep.copy_(ints(lengths))
        t.cuda.synchronize()
        graphs[1].replay() if captured else end()
        t.cuda.synchronize()
        assert n_free.item() == n_pages - sum(ref.pages(a, page) for a in lengths)


def test_prompt_rows_from_slots(rmi):
    """a packed prompt batch through the prep: slots in order make an fp16 pool's rows the prompt call's k and v"""
    t = torch()
    rng = np.random.default_rng(2)
    lens, n_kv, G, hd, page = [30, 1, 65], 2, 4, 256, 32
    n, nh = sum(lens), n_kv * G
    w3 = 2 * nh * hd + 2 * n_kv * hd
    x = rng.standard_normal((n, w3)).astype(np.float32)
    q3 = t.from_numpy(x).cuda()
    pos = np.concatenate([np.arange(m) for m in lens])
    pools = [t.zeros(3 * page, n_kv, hd, dtype=t.float16, device="cuda") for _ in range(2)]
    q, y = (t.empty(n, nh, hd, dtype=t.float16, device="cuda") for _ in range(2))
    rmi.attn_prep_paged(q3, w3, None, None, F16, pools[0], F16, pools[1], ints(np.arange(n)), ints(pos), q, nh, n_kv, hd, 64, rmi.ROPE_HALF, BASE, EPS, n,
                        page, 3)
    start = np.concatenate([[0], np.cumsum(lens)])
    scale = float(np.float32(hd ** -0.5))
    rmi.gqa_prompt_attn(q, nh * hd, pools[0], n_kv * hd, pools[1], n_kv * hd, ints(start), q3, w3, y, nh * hd, None, 0, 3, n, max(lens), nh, n_kv, hd, scale)
    hq, hk, hv, got = (a.double().cpu().numpy() for a in (q, pools[0], pools[1], y))
    gate = x[:, :2 * nh * hd].reshape(n, nh, 2, hd)[:, :, 1].astype(np.float64)
    for i, m in enumerate(lens):
        r = slice(start[i], start[i] + m)
        want, bound = ref.attention(hq[r], hk[r], hv[r], 0, scale, gate[r], 2.0 ** -11, 2.0 ** -11)
        assert (np.abs(got[r] - want) <= bound).all()
