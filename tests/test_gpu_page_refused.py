"""Requests that a plan refuses while they hold pages: what the prep and the attention do with their rows, and that ending or
retrying them loses no page and no history."""
import numpy as np
import pytest

from . import batch_ref as ref
from . import kv_ref
from .gpu_util import torch

pytestmark = pytest.mark.gpu
F16, I8, I4 = kv_ref.F16, kv_ref.I8, kv_ref.I4
PAGE, N_KV, G, HD, N_ROT, WIDTH, MOST, N_PAGES = 16, 2, 4, 128, 64, 16, 210, 14
EPS, BASE = 1e-6, 1e7

# rounds of (new tokens, status, how many of the positions in use then are kept: None all of them, 0 the request ends)
# 14 pages: 3 + 2 + 7 of them held after the first round
ENDS = [([40, 20, 100, 0], [0, 0, 0, 0], [None] * 4),
        ([60, 1, 1, 40], [2, 0, 0, 2], [0, None, None, None]),     # 4 more wanted, 2 left; refused while it holds 3, and ends
        ([0, 1, 1, 40], [0, 0, 0, 0], [None] * 4),                 # its pages serve another
        ([1, 200, -1, 1], [0, 2, 1, 0], [0] * 4)]                  # refused for want of pages, for its length; all end
RETRIES = [([40, 20, 100, 0], [0, 0, 0, 0], [None] * 4),
           ([60, 1, 1, 0], [2, 0, 0, 0], [None, None, 0, None]),   # refused; another one ends
           ([60, 13, 0, 5], [0, 0, 0, 0], [None] * 4),             # now it is served, behind its own 40 positions
           ([1, 1, 0, 1], [0, 0, 0, 0], [0] * 4)]


@pytest.fixture(scope="module")
def rmi():
    torch()
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def ints(x):
    return torch().tensor(np.asarray(x, np.int32), dtype=torch().int32, device="cuda")


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4)])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("split", [128, 256])
@pytest.mark.parametrize("rounds", [ENDS, RETRIES])
def test_refused_requests(rmi, kt, vt, captured, split, rounds):
    t = torch()
    rng = np.random.default_rng(31)
    n, nh = 4, N_KV * G
    w3, blocks_of = 2 * nh * HD + 2 * N_KV * HD, nh * HD // 32 * 36
    bytes_of = [ref.Pool(x, 1, PAGE, N_KV, HD, fill=0).raw.shape[1] for x in (kt, vt)]
    pools = [t.from_numpy(rng.integers(0, 256, (N_PAGES, b), dtype=np.uint8)).cuda() for b in bytes_of]
    table, free = ints(np.full((n, WIDTH), -1)), ints(rng.permutation(N_PAGES))
    n_free, n_left = ints([N_PAGES]), ints([0])
    past, count, keep, held = (ints([0] * n) for _ in range(4))
    row_start, kv_len, status = ints([0] * (n + 1)), ints([0] * n), ints([0] * n)
    slot, pos = ints([0] * MOST), ints([0] * MOST)
    q3 = t.zeros(MOST, w3, device="cuda")
    q, y = (t.zeros(MOST, nh, HD, dtype=t.float16, device="cuda") for _ in range(2))
    q8 = t.zeros(MOST, blocks_of, dtype=t.uint8, device="cuda")
    max_ctx, scale = WIDTH * PAGE, float(np.float32(HD ** -0.5))
    ws = t.empty(rmi.gqa_paged_workspace_bytes(MOST, max_ctx, nh, HD, split), dtype=t.uint8, device="cuda")

    def round_():
        rmi.page_plan(past, count, n, PAGE, N_PAGES, free, n_free, table, WIDTH, MOST, row_start, kv_len, slot, pos, n_left, status)
        rmi.attn_prep_paged(q3, w3, None, None, kt, pools[0], vt, pools[1], slot, pos, q, nh, N_KV, HD, N_ROT, rmi.ROPE_HALF, BASE, EPS, MOST, PAGE,
                            N_PAGES)
        rmi.gqa_paged_attn(q, kt, pools[0], vt, pools[1], table, WIDTH, row_start, kv_len, q3, w3, y, nh * HD, q8, blocks_of, ws, n, MOST, MOST,
                           max_ctx, nh, N_KV, HD, PAGE, N_PAGES, split, scale)

    def end():   # what a request holds: kv_len, or past where it was refused (kv_len alone would lose 3 pages of ENDS, 12 at the end)
        t.maximum(kv_len, past, out=held)
        rmi.page_trim(held, keep, n, PAGE, N_PAGES, table, WIDTH, n_left, free, n_free)

    graphs = None
    if captured:
        graphs = [t.cuda.CUDAGraph() for _ in range(2)]
        for g, f in zip(graphs, (round_, end)):
            with t.cuda.graph(g):
                f()
    lengths = [0] * n
    hist = [(np.zeros((0, N_KV, HD)), np.zeros((0, N_KV, HD))) for _ in range(n)]
    for counts, want_status, kept in rounds:
        past.copy_(ints(lengths)), count.copy_(ints(counts))
        x = rng.standard_normal((MOST, w3)).astype(np.float32)
        q3.copy_(t.from_numpy(x))
        q.fill_(float("nan"))   # rows that the prep leaves out
        y.fill_(77.0)
        q8.fill_(0xee)
        t.cuda.synchronize()
        graphs[0].replay() if captured else round_()
        t.cuda.synchronize()
        assert status.cpu().tolist() == want_status
        served = [s == 0 for s in want_status]
        total = [a + c if ok else 0 for a, c, ok in zip(lengths, counts, served)]
        assert kv_len.cpu().tolist() == total
        in_use = [max(a, b) for a, b in zip(total, lengths)]
        ids = [table[i, :ref.pages(m, PAGE)].cpu().tolist() for i, m in enumerate(in_use)]
        live = sum(ids, [])
        assert len(set(live)) == len(live) and n_left.item() == N_PAGES - len(live)
        got, blocks, held_q = y.double().cpu().numpy(), q8.cpu().numpy(), q.double().cpu().numpy()
        start = np.concatenate([[0], np.cumsum(np.maximum(counts, 0))])
        for i, c in enumerate(counts):
            rows = slice(start[i], start[i + 1])
            if not served[i]:
                assert (got[rows] == 0).all() and (blocks[rows] == 0).all() and np.isnan(held_q[rows]).all()
                continue
            if c == 0:
                continue
            k, v = x[rows, 2 * nh * HD:].reshape(c, 2, N_KV, HD).transpose(1, 0, 2, 3)
            k = ref.rotated(k, None, lengths[i] + np.arange(c), N_ROT, False, EPS, BASE)
            hist[i] = tuple(np.concatenate([old, kv_ref.held(new.astype(np.float32), type_)]) for old, new, type_ in zip(hist[i], (k, v), (kt, vt)))
            gate = x[rows, :2 * nh * HD].reshape(c, nh, 2, HD)[:, :, 1].astype(np.float64)
            want, bound = ref.attention(held_q[rows], *hist[i], lengths[i], scale, gate, 2.0 ** -11, 2.0 ** -11)
            assert (np.abs(got[rows] - want) <= bound).all(), f"request {i}"
        assert (got[start[-1]:] == 77.0).all() and (blocks[start[-1]:] == 0xee).all()
        lengths = [m if k is None else k for m, k in zip(in_use, kept)]
        hist = [(a[:m], b[:m]) for (a, b), m in zip(hist, lengths)]
        keep.copy_(ints(lengths))
        t.cuda.synchronize()
        graphs[1].replay() if captured else end()
        t.cuda.synchronize()
        still = [p for i, m in enumerate(lengths) for p in ids[i][:ref.pages(m, PAGE)]]
        back = free[:n_free.item()].cpu().tolist()
        assert sorted(back + still) == list(range(N_PAGES)), "every page is free or in use by one request"
    assert lengths == [0] * n and n_free.item() == N_PAGES
