"""Page plans, trims, reads and the prep with lengths, page ids and slots that are none: outputs between guards, against the plain
restatement where it says what they are."""
import numpy as np
import pytest

from . import batch_ref as ref
from . import kv_ref
from .gpu_util import torch

pytestmark = pytest.mark.gpu
F16, I8, I4 = kv_ref.F16, kv_ref.I8, kv_ref.I4
GUARD = 1 << 14   # elements on either side


@pytest.fixture(scope="module")
def rmi():
    torch()
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def ints(x):
    return torch().tensor(np.asarray(x, np.int64).astype(np.int32), dtype=torch().int32, device="cuda")


class Guarded:
    def __init__(self, values, guard):
        t = torch()
        values = values if isinstance(values, t.Tensor) else ints(values)
        self.guard, self.n = guard, values.numel()
        self.all = t.full((self.n + 2 * GUARD,), guard, dtype=values.dtype, device="cuda")
        self.t = self.all[GUARD:GUARD + self.n].view(values.shape)
        self.t.copy_(values)

    def check(self):
        t = torch()
        t.cuda.synchronize()
        assert bool((self.all[:GUARD] == self.guard).all()) and bool((self.all[GUARD + self.n:] == self.guard).all())


ODD = [0, 1, -1, 15, 16, 17, 100, 1000, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("n", [1, 5, 64, 300, 4096])
@pytest.mark.parametrize("page,width", [(16, 7), (256, 3)])
def test_plan_and_trim(rmi, n, page, width):
    rng = np.random.default_rng(n + page)
    for trial in range(6):
        n_pages, max_tok = int(rng.integers(1, 400)), int(rng.integers(1, 3000))
        odd = rng.random(n) < 0.3
        past = np.where(odd, rng.choice(ODD, n), rng.integers(0, width * page, n))
        count = np.where(rng.random(n) < 0.2, rng.choice(ODD, n), rng.integers(0, 20, n))
        n_free = int(rng.choice([-3, 0, n_pages // 2, n_pages, n_pages + 5, 2 ** 31 - 1]))
        table = np.where(rng.random((n, width)) < 0.2, rng.choice(ODD, (n, width)), rng.integers(0, n_pages, (n, width)))
        free = np.where(rng.random(n_pages) < 0.1, rng.choice(ODD, n_pages), rng.integers(0, n_pages, n_pages))
        out = [Guarded(np.full(k, -99), -1234567) for k in (n + 1, n, max_tok, max_tok, 1, n)]
        tab = Guarded(table, -1234567)
        rmi.page_plan(ints(past), ints(count), n, page, n_pages, ints(free), ints([n_free]), tab.t, width, max_tok, *(x.t for x in out))
        for x in out + [tab]:
            x.check()
        want = ref.plan(past, count, page, n_pages, free, min(max(n_free, 0), n_pages), table, max_tok)
        got = [x.t.cpu().numpy() for x in out]
        for i in (0, 1, 2, 5):
            assert np.array_equal(got[i], want[(0, 1, 2, 3, 4, 5)[i]]), i
        assert got[4][0] == want[4] and np.array_equal(tab.t.cpu().numpy(), want[6])
        keep = np.where(rng.random(n) < 0.3, rng.choice(ODD, n), rng.integers(0, width * page + 40, n))
        fr, left = Guarded(free, -1234567), Guarded([-99], -1234567)
        rmi.page_trim(ints(past), ints(keep), n, page, n_pages, ints(table), width, ints([n_free]), fr.t, left.t)
        fr.check(), left.check()
        at, after = ref.trim(past, keep, page, n_pages, table, min(max(n_free, 0), n_pages), free)
        assert left.t.item() == at and fr.t.cpu().tolist() == list(after)


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4), (I4, I8)])
@pytest.mark.parametrize("hd,page", [(128, 16), (256, 64)])
def test_prep_and_read(rmi, kt, vt, hd, page):
    t = torch()
    rng = np.random.default_rng(hd + kt)
    n, n_kv, nh, n_pages = 60, 2, 4, 3
    slots = n_pages * page
    slot = np.where(rng.random(n) < 0.5, rng.choice([-1, -2 ** 31, slots, slots + 1, 2 ** 31 - 1, -slots], n), -1)
    inside = rng.permutation(n)[:min(n, slots) // 2]
    slot[inside] = rng.permutation(slots)[:len(inside)]
    used = (slot >= 0) & (slot < slots)
    pos = rng.choice([0, 1, 17, 4000, 2 ** 30, 2 ** 31 - 1, -5], n)
    width = 2 * nh * hd + 2 * n_kv * hd
    x = rng.standard_normal((n, width)).astype(np.float32)
    raw = [ref.Pool(ty, n_pages, page, n_kv, hd, rng=rng).raw for ty in (kt, vt)]
    pools = [Guarded(t.from_numpy(r).cuda(), 0x3b) for r in raw]
    q = Guarded(t.full((n, nh, hd), 77.0, dtype=t.float16, device="cuda"), 77.0)
    rmi.attn_prep_paged(t.from_numpy(x).cuda(), width, None, None, kt, pools[0].t, vt, pools[1].t, ints(slot), ints(pos), q.t, nh, n_kv, hd, 64, rmi.ROPE_HALF,
                        1e7, 1e-6, n, page, n_pages)
    for g in pools + [q]:
        g.check()
    written = (q.t != 77.0).flatten(1).any(1).cpu().numpy()
    assert np.array_equal(written, used)
    v = x[:, 2 * nh * hd:].reshape(n, 2, n_kv, hd)[:, 1]
    for ty, pool, before, rows in ((kt, pools[0], raw[0], None), (vt, pools[1], raw[1], kv_ref.held(v, vt))):
        after = pool.t.cpu().numpy()
        mine = np.zeros((n_pages, page), bool)
        mine.reshape(-1)[slot[used]] = True
        for p in range(n_pages):
            touched = np.zeros(after.shape[1], bool)
            for s in np.nonzero(mine[p])[0]:   # the bytes of position s: those of the first s + 1 without those of the first s
                touched |= ref.kv_ref_mask(ty, s + 1, page, n_kv, hd) & ~ref.kv_ref_mask(ty, s, page, n_kv, hd)
            assert np.array_equal(after[p][~touched], before[p][~touched])
        out = Guarded(t.full((n, n_kv * hd), 55.0, dtype=t.float32, device="cuda"), 55.0)
        rmi.kv_page_read(ty, pool.t, ints(slot), out.t, n_kv * hd, n, n_kv, hd, page, n_pages)
        out.check()
        got = out.t.cpu().numpy().reshape(n, n_kv, hd)
        assert (got[~used] == 0).all() and (rows is None or np.array_equal(got[used], rows[used].astype(np.float32)))
