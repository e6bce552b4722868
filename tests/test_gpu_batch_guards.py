"""Outputs and workspaces of the batch attention between guards: row starts and lengths that are none write nothing outside a call's
rows, what they do name is the formula's."""
import numpy as np
import pytest

from . import batch_exact as exact
from . import batch_ref as ref
from . import kv_ref
from .gpu_util import torch
from .test_gpu_batch_attn import Batch, ints

pytestmark = pytest.mark.gpu
F16, I8, I4 = kv_ref.F16, kv_ref.I8, kv_ref.I4
GUARD = 1 << 16   # bytes on either side
FAR = 2 ** 31 - 1
# starts beyond the call, negative, descending; rows of no request before the first one (a join then finds none that begins at or
# before them), between and behind
STARTS = [[0, 1, 10 ** 9, 10 ** 9], [-5, -9, 3, 2], [7, 3, 1, 0], [FAR, -2 ** 31, FAR, 5], [0, 25, 0, 25], [-2 ** 31, 0, 0, FAR], [4, 4, 9, 9]]


@pytest.fixture(scope="module")
def rmi():
    torch()
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


class Guarded:
    """a tensor inside a larger one, all of it filled with a byte"""

    def __init__(self, shape, dtype, byte):
        t = torch()
        self.byte, self.n = byte, int(np.prod(shape)) * t.empty(0, dtype=dtype).element_size()
        self.all = t.full((self.n + 2 * GUARD,), byte, dtype=t.uint8, device="cuda")
        self.raw = self.all[GUARD:GUARD + self.n]
        self.t = self.raw.view(dtype).view(shape)

    def check(self):
        assert bool((self.all[:GUARD] == self.byte).all()) and bool((self.all[GUARD + self.n:] == self.byte).all())

    def rows(self):
        """which of the first dimension's rows have been written"""
        return (self.raw.view(self.t.shape[0], -1) != self.byte).any(1).cpu().numpy()


def ranges(start, ntok, most):
    """rows of each request, as the header has them: cut to the call's; none past the bound of new tokens"""
    out = []
    for a, e in zip(start, start[1:]):
        a = min(max(a, 0), ntok)
        n = min(max(e, a), ntok) - a
        out.append((a, n if n <= most else 0))
    return out


def named(spans, n):
    used = np.zeros(n, np.int64)
    for a, m in spans:
        used[a:a + m] += 1
    return used


@pytest.mark.parametrize("kt,vt", [(F16, F16), (I8, I4)])
@pytest.mark.parametrize("most", [20, 64])
@pytest.mark.parametrize("split,max_ctx", [(128, 270), (128, 2000), (2048, 2000)])   # a join of three chunks, one of 16, none
def test_paged(rmi, kt, vt, most, split, max_ctx):
    t = torch()
    rng = np.random.default_rng(4)
    lens = [(100, 1), (250, 20), (70, 2)]
    for G, page in ((4, 32), (1, 16)):
        b = Batch(rng, lens, kt, vt, 2, G, 128, page)
        assert b.ntok == 25
        total, nh, hd = [101, 270, 72], b.nh, b.hd
        for start in STARTS:
            for length in (total, [101, -7, 72], [FAR, 270, 0]):
                y, q8 = Guarded((b.ntok, nh, hd), t.float16, 0x5c), Guarded((b.ntok, nh * hd // 32 * 36), t.uint8, 0xee)
                ws = Guarded((rmi.gqa_paged_workspace_bytes(b.ntok, max_ctx, nh, hd, split),), t.uint8, 0xff)
                pools = [t.from_numpy(x.raw).cuda() for x in (b.k, b.v)]
                rmi.gqa_paged_attn(b.tq, kt, pools[0], vt, pools[1], ints(b.table), b.width, ints(np.array(start, np.int64)), ints(np.array(length, np.int64)),
                                   t.from_numpy(b.gate).cuda(), 2 * nh * hd, y.t, nh * hd, q8.t, q8.t.shape[1], ws.t, 3, b.ntok, most, max_ctx, nh, 2, hd, page,
                                   b.n_pages, split, b.scale)
                t.cuda.synchronize()
                for x in (y, q8, ws):
                    x.check()
                spans = [(a, n if m <= max_ctx else 0) for (a, n), m in zip(ranges(start, b.ntok, most), length)]
                used = named(spans, b.ntok)
                for x in (y, q8):
                    written = x.rows()
                    assert not written[used == 0].any()
                    if split > 128 or start == sorted(start):   # a join looks for a row's request among starts that ascend
                        assert written[used > 0].all()
                if start != sorted(start) and split == 128:
                    continue
                for i, (a, n) in enumerate(spans):
                    rows = [r for r in range(a, a + n) if used[r] == 1]   # rows of two requests are either's
                    if not rows:
                        continue
                    pos = t.tensor([length[i] - n + r - a for r in rows], device="cuda")
                    before = pos < 0
                    got = y.t[rows].double()
                    assert bool((got[before] == 0).all())
                    held = [t.from_numpy(x).cuda() for x in b.held(i)]
                    if bool((pos >= len(held[0])).any()):
                        continue
                    live = t.tensor(rows, device="cuda")[~before]
                    if len(live):
                        want, bound = exact.attention(b.tq[live].double(), *held, pos[~before], b.scale, 2.0 ** -11, 2.0 ** -11,
                                                      t.from_numpy(b.gate[live.cpu().numpy(), :, 1].astype(np.float64)).cuda())
                        assert exact.outside(got[~before], want, bound) == 0


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("ntok,n_req,n_kv,G", [(25, 3, 1, 8), (143, 3, 1, 8), (600, 70, 2, 8), (268, 3, 8, 64)])
def test_prompts(rmi, name, ntok, n_req, n_kv, G):
    """the forms of few tiles, of four waves and of eight (by the heads), the long prompts' requests among those that are none"""
    t = torch()
    hd, dtype, nh = 128, getattr(t, name), n_kv * G
    rng = np.random.default_rng(ntok)
    q, k, v = (t.from_numpy(rng.standard_normal((ntok, h, hd)).astype(np.float32)).to(dtype).cuda() for h in (nh, n_kv, n_kv))
    scale = float(np.float32(hd ** -0.5))
    for start in STARTS:
        start = start + [ntok] * (n_req - 3)   # what follows is empty, or the rest
        for most in (ntok, 20):
            y, q8 = Guarded((ntok, nh, hd), dtype, 0x5c), Guarded((ntok, nh * hd // 32 * 36), t.uint8, 0xee)
            rmi.gqa_prompt_attn(q, nh * hd, k, n_kv * hd, v, n_kv * hd, ints(np.array(start, np.int64)), None, 0, y.t, nh * hd, q8.t, q8.t.shape[1], n_req,
                                ntok, most, nh, n_kv, hd, scale)
            t.cuda.synchronize()
            for x in (y, q8):
                x.check()
            spans = ranges(start, ntok, most)
            used = named(spans, ntok)
            once = used.max() <= 1   # overlapping requests may have more tiles than the launch is made for
            for x in (y, q8):
                written = x.rows()
                assert not written[used == 0].any()
                if once:
                    assert written[used > 0].all()
            if not once:
                continue
            for a, n in spans:
                rows = sorted({a + r for e in (0, 1, 8, 16, 31) for r in (e, n - 1 - e) if 0 <= r < n})
                if rows:
                    pos = t.tensor(rows, device="cuda") - a
                    heads = [0, nh - 1]
                    want, bound = exact.attention(q[rows][:, heads].double(), k[a:a + n, [0, n_kv - 1]].double(), v[a:a + n, [0, n_kv - 1]].double(), pos, scale,
                                                  ref.HALF_STEP[name], ref.HALF_STEP[name])
                    assert exact.outside(y.t[rows][:, heads].double(), want, bound) == 0
