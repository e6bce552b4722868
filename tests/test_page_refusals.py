"""Argument checks of the calls on pages and packed prompts, before any device work (CPU)."""
import ctypes

import pytest


def at(n):
    return ctypes.c_void_p(n << 26)   # aligned, far apart, never dereferenced: validation fails first


NULL = None


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def off(p, n):
    return ctypes.c_void_p(p.value + n)


def test_plan(rmi):
    def call(past=at(1), count=at(2), n=4, page=64, n_pages=100, free=at(3), n_free=at(4), table=at(5), width=8, max_tok=64, row=at(6),
             kv=at(7), slot=at(8), pos=at(9), left=at(10), status=at(11)):
        rmi._call("rmi_page_plan", past, count, n, page, n_pages, free, n_free, table, width, max_tok, row, kv, slot, pos, left, status, None)

    for bad in ({"n": 0}, {"n": 4097}, {"page": 0}, {"page": 8}, {"page": 48}, {"page": 512}, {"n_pages": 0}, {"n_pages": 2 ** 31 - 1}, {"width": 0},
                {"width": 2 ** 30}, {"max_tok": 0}, {"max_tok": 2 ** 30 + 1}, {"past": NULL}, {"count": NULL}, {"free": NULL}, {"n_free": NULL},
                {"table": NULL}, {"row": NULL}, {"kv": NULL}, {"slot": NULL}, {"pos": off(at(9), 2)}, {"left": NULL}, {"status": NULL},
                {"left": at(4)}, {"kv": at(1)}, {"slot": at(9)}, {"pos": off(at(8), 4 * 63)}, {"status": off(at(6), 16)}, {"table": off(at(3), 396)},
                {"row": off(at(2), 12)}):
        with pytest.raises(ValueError, match="page_plan"):
            call(**bad)


def test_trim(rmi):
    def call(length=at(1), keep=at(2), n=4, page=64, n_pages=100, table=at(3), width=8, n_free=at(4), free=at(5), out=at(6)):
        rmi._call("rmi_page_trim", length, keep, n, page, n_pages, table, width, n_free, free, out, None)

    for bad in ({"n": 0}, {"n": 4097}, {"page": 24}, {"n_pages": -1}, {"width": 0}, {"length": NULL}, {"keep": NULL}, {"table": off(at(3), 1)},
                {"n_free": NULL}, {"free": NULL}, {"out": NULL}, {"out": at(4)}, {"free": off(at(3), 124)}, {"out": off(at(5), 396)}, {"free": at(1)}):
        with pytest.raises(ValueError, match="page_trim"):
            call(**bad)


def test_rows(rmi):
    def call(type_=1, pool=at(1), slot=at(3), out=at(4), f16=1, stride=1024, n=5, n_kv=4, hd=256, page=64, n_pages=10):
        rmi._call("rmi_kv_page_read", type_, pool, slot, out, f16, stride, n, n_kv, hd, page, n_pages, None)

    call(n=0)
    for bad in ({"type_": 3}, {"n": -1}, {"stride": 1023}, {"n_kv": 0}, {"hd": 64}, {"page": 40}, {"n_pages": 0}, {"pool": off(at(1), 8)}, {"slot": NULL},
                {"out": NULL}, {"out": off(at(4), 1)}, {"out": off(at(4), 2), "f16": 0}, {"out": off(at(1), 32)}, {"out": off(at(3), 16)}):
        with pytest.raises(ValueError, match="kv_page_read"):
            call(**bad)


def test_prep(rmi):
    def call(q3=at(1), stride=10240, qn=at(2), kn=at(3), kt=1, k=at(4), vt=2, v=at(5), slot=at(6), pos=at(7), qt=0, q=at(8), nh=16, nkv=4, hd=256,
             n_rot=64, base=1e7, factor=1.0, orig=0.0, pairs=0, n=3, page=64, n_pages=10, rope=True):
        r = rmi.RopeParams(base, factor, orig, 1.0, 1.0, 32.0, 1.0)
        rmi._call("rmi_attn_prep_paged", q3, stride, qn, kn, kt, k, vt, v, slot, pos, qt, q, nh, nkv, hd, n_rot, ctypes.byref(r) if rope else None, pairs,
                  1e-6, n, page, n_pages, None)

    for bad in ({"kt": 3}, {"vt": -1}, {"qt": 2}, {"nh": 15}, {"nh": 0}, {"nkv": 0}, {"hd": 64}, {"n_rot": 63}, {"n_rot": 258}, {"n_rot": -2}, {"base": 1.0},
                {"base": float("nan")}, {"factor": 2.0}, {"pairs": 2}, {"n": 0}, {"page": 65}, {"n_pages": 0}, {"rope": False}, {"q3": NULL},
                {"qn": off(at(2), 2)}, {"k": NULL}, {"v": off(at(5), 8)}, {"slot": NULL}, {"pos": NULL}, {"q": off(at(8), 8)}, {"q": NULL},
                {"v": at(4)}, {"q": at(1)}, {"q": off(at(1), 2 * 40960 + 40944)}, {"k": off(at(6), 0)}, {"q": off(at(4), 1024)}, {"v": at(2)}):
        with pytest.raises(ValueError, match="attn_prep_paged"):
            call(**bad)


def test_paged_attention(rmi):
    def call(qt=0, q=at(1), kt=1, k=at(2), vt=1, v=at(3), table=at(4), width=8, row=at(5), kv=at(6), gate=at(7), gs=8192, y=at(8), ys=4096, q8=at(9),
             q8s=4608, ws=at(10), n=4, ntok=9, new=5, ctx=500, nh=16, nkv=4, hd=256, page=64, n_pages=10, split=128, scale=0.0625):
        rmi._call("rmi_gqa_paged_attn", qt, q, kt, k, vt, v, table, width, row, kv, gate, gs, y, ys, q8, q8s, ws, n, ntok, new, ctx, nh, nkv, hd, page,
                  n_pages, split, scale, None)

    for bad in ({"qt": 2}, {"kt": 0}, {"kt": 2, "vt": 1}, {"vt": 0}, {"kt": 7}, {"n": 0}, {"n": 4097}, {"ntok": 0}, {"ntok": 2 ** 24 + 1}, {"new": 0},
                {"ctx": 0}, {"ctx": 2 ** 30 + 1, "split": 2 ** 30}, {"nh": 15}, {"nh": 4 * 65, "nkv": 4}, {"nkv": 0}, {"hd": 64}, {"page": 100}, {"n_pages": 0},
                {"width": 0}, {"split": 0}, {"split": 100}, {"split": -128}, {"ctx": 2 ** 20}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
                {"scale": float("inf")}, {"q": NULL}, {"q": off(at(1), 8)}, {"k": NULL}, {"v": off(at(3), 4)}, {"table": NULL}, {"row": NULL}, {"kv": NULL},
                {"gate": off(at(7), 2)}, {"y": NULL, "q8": NULL}, {"y": off(at(8), 4)}, {"ys": 4095}, {"ys": 4098}, {"ys": 4092}, {"q8s": 4604}, {"q8s": 4610},
                {"q8": off(at(9), 2)}, {"ws": NULL}, {"ws": off(at(10), 4)}, {"y": at(1)}, {"y": at(2)}, {"y": off(at(3), 16)}, {"q8": at(8)}, {"ws": at(2)},
                {"ws": at(8)}, {"y": off(at(7), 1024)}, {"y": at(4)}, {"q8": at(6)}, {"ws": at(5)}, {"y": off(at(10), 16)}):
        with pytest.raises(ValueError, match="gqa_paged_attn"):
            call(**bad)


def test_prompt_attention(rmi):
    def call(t=0, q=at(1), qs=4096, k=at(2), ks=1024, v=at(3), vs=1024, row=at(5), gate=at(7), gs=8192, y=at(8), ys=4096, q8=at(9), q8s=4608, n=4, ntok=9,
             longest=5, nh=16, nkv=4, hd=256, scale=0.0625):
        rmi._call("rmi_gqa_prompt_attn", t, q, qs, k, ks, v, vs, row, gate, gs, y, ys, q8, q8s, n, ntok, longest, nh, nkv, hd, scale, None)

    for bad in ({"t": 2}, {"n": 0}, {"ntok": 0}, {"longest": 0}, {"nh": 10}, {"hd": 192}, {"scale": 0.0}, {"qs": 4092}, {"qs": 4088}, {"ks": 1020}, {"ks": 1016},
                {"vs": 1025}, {"ks": 2 ** 25 + 8}, {"vs": 2 ** 25 + 8}, {"n": 4097}, {"ntok": 2 ** 24 + 1}, {"scale": float("nan")},
                {"ntok": 2 ** 24, "longest": 2 ** 24, "nh": 64 * 64, "nkv": 64, "qs": 64 * 64 * 256, "ks": 2 ** 14, "vs": 2 ** 14, "ys": 2 ** 20, "q8s": 2 ** 21, "gate": NULL, "k": at(2 ** 24), "v": at(2 ** 25), "y": at(2 ** 26), "q8": NULL, "hd": 256},
                {"q": NULL}, {"k": off(at(2), 8)}, {"v": NULL}, {"row": NULL}, {"gate": off(at(7), 1)}, {"y": NULL, "q8": NULL},
                {"y": off(at(8), 4)}, {"ys": 4094}, {"q8s": 4000}, {"y": at(1)}, {"y": at(3)}, {"q8": at(2)}, {"y": at(9)}, {"q8": off(at(7), 1024)},
                {"y": at(5)}):
        with pytest.raises(ValueError, match="gqa_prompt_attn"):
            call(**bad)


def test_split_and_workspace(rmi):
    assert rmi.gqa_paged_split(4096, 4096, 1, 1, 1, 16, 4, 256) % 128 == 0
    assert rmi.gqa_paged_workspace_bytes(3, 500, 16, 256, 512) == 16
    assert rmi.gqa_paged_workspace_bytes(3, 500, 16, 256, 128) == 4 * 3 * 16 * 258 * 4
    for ctx in (1, 127, 4096, 65536, 1 << 20, 1 << 30):
        for reqs, new in ((1, 1), (64, 1), (1, 999), (4096, 4)):
            s = rmi.gqa_paged_split(min(ctx * reqs, 2 ** 40), ctx, reqs, reqs * new, new, 16, 4, 256)
            assert s % 128 == 0 and -(-ctx // s) <= 1024
            assert rmi.gqa_paged_workspace_bytes(reqs * new, ctx, 16, 256, s) > 0
    for bad in ((0, 1, 1, 1, 1, 16, 4, 256), (1, 0, 1, 1, 1, 16, 4, 256), (1, 1, 0, 1, 1, 16, 4, 256), (1, 1, 1, 0, 1, 16, 4, 256), (1, 1, 1, 1, 0, 16, 4, 256),
                (1, 1, 1, 1, 1, 15, 4, 256), (1, 1, 1, 1, 1, 16, 4, 64)):
        with pytest.raises(ValueError, match="gqa_paged_split"):
            rmi.gqa_paged_split(*bad)
    for bad in ((0, 500, 16, 256, 128), (3, 0, 16, 256, 128), (3, 500, 0, 256, 128), (3, 500, 16, 100, 128), (3, 500, 16, 256, 100), (3, 2 ** 20, 16, 256, 128)):
        with pytest.raises(ValueError, match="gqa_paged_workspace_bytes"):
            rmi.gqa_paged_workspace_bytes(*bad)


def test_bindings_check_types(rmi):
    torch = pytest.importorskip("torch")
    f32, f16, bf16, i32, i64 = (torch.zeros(8, dtype=d) for d in (torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.int64))
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        rmi.gqa_prompt_attn(f32, 8, f16, 8, f16, 8, i32, None, 0, f16, 8, None, 0, 1, 1, 1, 1, 1, 128, 1.0)
    with pytest.raises(ValueError, match="one type"):
        rmi.gqa_prompt_attn(f16, 8, bf16, 8, f16, 8, i32, None, 0, f16, 8, None, 0, 1, 1, 1, 1, 1, 128, 1.0)
    with pytest.raises(ValueError, match="int32"):
        rmi.page_trim(i64, i32, 1, 16, 1, i32, 1, i32, i32, i32)
    with pytest.raises(ValueError, match="current GPU"):
        rmi.page_trim(i32, i32, 1, 16, 1, i32, 1, i32, i32, i32)
    with pytest.raises(ValueError, match="float32"):
        rmi.attn_prep_paged(f16, 8, None, None, 0, f16, 0, f16, i32, i32, f16, 1, 1, 128, 0, 0, 1e4, 1e-6, 1, 16, 1)
    with pytest.raises(ValueError, match="one type"):
        rmi.gqa_paged_attn(f16, 0, f16, 0, f16, i32, 1, i32, i32, None, 0, bf16, 8, None, 0, None, 1, 1, 1, 1, 1, 1, 128, 16, 1, 128, 1.0)
