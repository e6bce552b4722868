"""Argument checks of the quantised-cache, tree-attention and logit entry points, before any device work (CPU)."""
import ctypes

import pytest

FAKE = ctypes.c_void_p(1 << 20)
OFF8 = ctypes.c_void_p((1 << 20) + 8)
OFF4 = ctypes.c_void_p((1 << 20) + 4)
FAR = ctypes.c_void_p(1 << 30)
ODD = ctypes.c_void_p((1 << 20) + 1)


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


def test_cache_bytes(rmi):
    assert rmi.kv_cache_bytes(rmi.KV_F16, 100, 4, 256) == 100 * 4 * 512
    assert rmi.kv_cache_bytes(rmi.KV_I8, 100, 4, 256) == 100 * 4 * (256 + 8)
    assert rmi.kv_cache_bytes(rmi.KV_I4, 100, 3, 128) == 100 * 3 * (64 + 4)
    assert rmi.kv_cache_bytes(rmi.KV_I8, 1 << 30, 8, 256) == (1 << 33) * 264
    for bad in ((3, 100, 4, 256), (-1, 100, 4, 256), (1, 0, 4, 256), (1, 100, 0, 256), (1, 100, 4, 64), (1, 100, 4, 192),
                (1, (1 << 30) + 1, 1, 128), (1, 100, 65536, 128)):
        with pytest.raises(ValueError):
            rmi.kv_cache_bytes(*bad)


@pytest.mark.parametrize("name", ["rmi_kv_write", "rmi_kv_read"])
def test_rows(rmi, name):
    def call(type_=1, rows=FAKE, f16=0, stride=1024, cache=FAKE, first=0, n=0, n_kv=4, hd=256, max_ctx=100):
        a = (rows, f16, stride, cache) if name == "rmi_kv_write" else (cache, rows, f16, stride)
        rmi._call(name, type_, *a, first, n, n_kv, hd, max_ctx, None)

    call()
    call(first=100)
    for bad in ({"type_": 3}, {"stride": 1023}, {"first": -1}, {"n": -1}, {"n": 101}, {"first": 1, "n": 100}, {"first": 101},
                {"first": 2 ** 31 - 1, "n": 1}, {"n_kv": 0}, {"hd": 100}, {"max_ctx": 0}, {"rows": None}, {"cache": None}, {"cache": OFF8},
                {"rows": ODD, "f16": 1}, {"rows": ctypes.c_void_p((1 << 20) + 2)}):
        with pytest.raises(ValueError, match="invalid"):
            call(**bad) if "type_" not in bad else call(**bad)


def test_compact(rmi):
    def call(type_=1, ptrs=(1 << 20,), n=None, pos=FAKE, path=FAKE, count=FAKE, max_path=4, n_kv=4, hd=256, max_ctx=100, null=False):
        arr = (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs)
        rmi._call("rmi_kv_compact", type_, None if null else arr, len(ptrs) if n is None else n, pos, path, count, max_path, n_kv, hd,
                  max_ctx, None)

    for bad in ({"type_": 7}, {"n": 0}, {"ptrs": (1 << 20,) * 65}, {"max_path": 0}, {"max_path": 65}, {"n_kv": 0}, {"hd": 64}, {"max_ctx": 0},
                {"null": True}, {"pos": None}, {"path": None}, {"count": None}, {"pos": ODD}, {"ptrs": (1 << 20, None)},
                {"ptrs": (1 << 20, 1 << 22, 1 << 20)}, {"ptrs": ((1 << 20) + 16, 1 << 20)},
                {"ptrs": ((1 << 20) + 8,)}):
        with pytest.raises(ValueError, match="kv_compact"):
            call(**bad)


def test_prep_axes(rmi):
    def call(q3=FAKE, qn=FAKE, kn=FAKE, ktype=1, k=FAKE, vtype=1, v=FAR, pos=FAKE, axis=FAKE, qout=FAKE, nh=16, nkv=4, hd=256, n_rot=64,
             base=1e7, factor=1.0, orig=0.0, sec=(12, 10, 10), inter=1, ntok=1, max_ctx=100, rope=True, axes=True):
        r = rmi.RopeParams(base, factor, orig, 1.0, 1.0, 32.0, 1.0)
        x = rmi.RopeAxes((ctypes.c_int * 3)(*sec), inter)
        rmi._call("rmi_attn_prep_axes", q3, 10240, qn, kn, ktype, k, vtype, v, pos, axis, qout, nh, nkv, hd, n_rot,
                  ctypes.byref(r) if rope else None, ctypes.byref(x) if axes else None, 1e-6, ntok, max_ctx, None)

    for bad in ({"ktype": 3}, {"vtype": -1}, {"nh": 15}, {"nh": 0}, {"nkv": 0}, {"hd": 192}, {"n_rot": 63}, {"n_rot": 258}, {"n_rot": -2},
                {"base": 1.0}, {"base": float("nan")}, {"factor": 2.0}, {"sec": (11, 10, 10)}, {"sec": (34, -1, -1)}, {"sec": (2 ** 31 - 1, 0, 0)},
                {"sec": (8, 12, 12)}, {"sec": (10, 10, 12)}, {"ntok": 0}, {"ntok": 101}, {"max_ctx": 0}, {"rope": False}, {"axes": False},
                {"q3": None}, {"qn": None}, {"kn": None}, {"k": None}, {"v": OFF4}, {"pos": None}, {"axis": ODD}, {"qout": None},
                {"v": FAKE}, {"k": FAR, "v": ctypes.c_void_p((1 << 30) + 1600)}):
        with pytest.raises(ValueError, match="attn_prep_axes"):
            call(**bad)


def test_tree_attention(rmi):
    def call(q=FAKE, ktype=1, k=FAKE, vtype=1, v=FAKE, pos=FAKE, masks=FAKE, gate=FAKE, y=FAKE, ys=4096, q8=FAKE, q8s=4608, ws=FAKE, nh=16, nkv=4, hd=256,
             ntok=8, max_ctx=1000, nsub=1):
        rmi._call("rmi_gqa_tree_decode", q, ktype, k, vtype, v, pos, masks, gate, 10240, y, ys, q8, q8s, ws, nh, nkv, hd, ntok, max_ctx, nsub,
                  0.0625, None)

    for bad in ({"ktype": 3}, {"vtype": 9}, {"ktype": 0}, {"vtype": 0}, {"ktype": 2, "vtype": 1}, {"nh": 15}, {"nh": 0}, {"nkv": 0},
                {"nh": 260}, {"hd": 64}, {"ntok": 0}, {"ntok": 65}, {"ntok": 1025, "masks": None, "max_ctx": 5000}, {"ntok": 9, "max_ctx": 8},
                {"max_ctx": 0}, {"nsub": 0}, {"nsub": -1}, {"nsub": 1 << 24}, {"nsub": 1 << 25}, {"nsub": (1 << 25) + 1}, {"nsub": 1, "max_ctx": 128 * 2048 + 1}, {"q": None}, {"q": OFF8}, {"k": None},
                {"v": OFF4}, {"pos": None}, {"masks": OFF4}, {"gate": ODD}, {"y": None, "q8": None}, {"y": ODD}, {"q8": ODD}, {"q8s": 4609},
                {"ys": 4095}, {"ys": -4096}, {"q8s": 4604}, {"ws": None}, {"ws": OFF8}):
        with pytest.raises(ValueError, match="gqa_tree_decode"):
            call(**bad)


def test_tree_plan(rmi):
    for ctx in (1, 127, 128, 5000, 65536, 1 << 20):
        for ntok in (1, 8, 64, 999):
            split = rmi.gqa_tree_nsub(ctx, 16, 4, 256, ntok)
            nsub = split & (rmi.TREE_SHORT - 1)
            assert split == nsub or split == nsub + rmi.TREE_SHORT
            assert 1 <= nsub <= max(6, -(-ctx // 128)) and -(-ctx // (128 * nsub)) <= 2048
            assert rmi.gqa_tree_workspace_bytes(ctx, 16, 4, 256, ntok, split) > 0
    for bad in ((0, 16, 4, 256, 1), (100, 15, 4, 256, 1), (100, 16, 4, 64, 1), (100, 16, 4, 256, 0), (100, 16, 4, 256, 1025)):
        with pytest.raises(ValueError):
            rmi.gqa_tree_nsub(*bad)
        with pytest.raises(ValueError):
            rmi.gqa_tree_workspace_bytes(*bad, 1)
    with pytest.raises(ValueError):
        rmi.gqa_tree_workspace_bytes(100, 16, 4, 256, 1, 0)
    for bad in (rmi.TREE_SHORT, 2 * rmi.TREE_SHORT, 2 * rmi.TREE_SHORT + 1, 2 ** 31 - 1):
        with pytest.raises(ValueError):
            rmi.gqa_tree_workspace_bytes(100, 16, 4, 256, 1, bad)
    with pytest.raises(ValueError):
        rmi.gqa_tree_workspace_bytes(128 * 2048 + 1, 16, 4, 256, 1, 1)
    with pytest.raises(ValueError):
        rmi.gqa_tree_workspace_bytes(128 * 2048 + 1, 16, 4, 256, 1, 1 + rmi.TREE_SHORT)


def test_logits(rmi):
    def call(x=FAKE, n=1000, ncols=2, cs=1000, out=OFF8, os=1000, hist=FAKE, hl=FAKE, mh=10, draft=FAKE, masks=FAKE, nd=2, rep=1.0, ids=FAKE,
             vals=FAKE, nb=3, allow=FAKE, als=32, pen=True):
        p = rmi.Penalties(rep, 0.0, 0.0, 0)
        rmi._call("rmi_logits_process", x, n, ncols, cs, out, os, hist, hl, mh, draft, masks, nd, ctypes.byref(p) if pen else None, ids, vals,
                  nb, allow, als, None)

    for bad in ({"n": 0}, {"n": 2 ** 31 - 1}, {"ncols": 0}, {"ncols": 65}, {"cs": 999}, {"os": 999}, {"mh": -1}, {"nd": -1}, {"nd": 65},
                {"nb": -1}, {"rep": 0.0}, {"rep": -1.0}, {"rep": float("nan")}, {"pen": False}, {"als": 31}, {"out": FAKE, "os": 1001},
                {"x": None}, {"out": None}, {"x": ODD}, {"hist": None}, {"hl": None}, {"draft": None}, {"masks": None}, {"masks": OFF4},
                {"ids": None}, {"vals": None}, {"allow": ODD}):
        with pytest.raises(ValueError, match="logits_process"):
            call(**bad)


def test_bindings_refuse_host_tensors_and_other_types(rmi):
    import torch
    x, i = torch.zeros(4096), torch.zeros(4, dtype=torch.int32)
    b = torch.zeros(1 << 20, dtype=torch.uint8)
    for f in (lambda: rmi.kv_write(rmi.KV_I8, x, 1024, b, 0, 1, 4, 256, 100),
              lambda: rmi.kv_read(rmi.KV_I8, b, x, 1024, 0, 1, 4, 256, 100),
              lambda: rmi.kv_compact(rmi.KV_I8, [b], i, i, i, 1, 4, 256, 100),
              lambda: rmi.gqa_tree_decode(x, 1, b, 1, b, i, None, None, 0, x, 4096, None, 0, b, 16, 4, 256, 1, 100, 1, 0.06),
              lambda: rmi.attn_prep_axes(x, 6144, x, x, 1, b, 1, b, i, None, x, 16, 4, 256, 64, 1e6, 1.0, 0.0, (12, 10, 10), True, 1e-6, 1, 100),
              lambda: rmi.logits_process(x, 100, 1, 100, x, 100, None, None, 0),
              lambda: rmi.logits_process(x, 100, 1, 100, x, 100, None, None, 0, stream=1)):
        with pytest.raises(ValueError, match="current GPU"):
            f()
    for t in (torch.bfloat16, torch.float64, torch.uint8):
        with pytest.raises(ValueError, match="float32 or float16"):
            rmi.kv_write(rmi.KV_I8, x.to(t), 1024, b, 0, 1, 4, 256, 100)
        with pytest.raises(ValueError, match="float32 or float16"):
            rmi.kv_read(rmi.KV_I8, b, x.to(t), 1024, 0, 1, 4, 256, 100)


def test_launches_stay_in_32_bit_work_items(rmi):
    with pytest.raises(ValueError, match="too many rows"):
        rmi._call("rmi_kv_read", 2, FAKE, FAR, 1, 64 * 256, 0, 1 << 22, 64, 256, 1 << 22, None)
    with pytest.raises(ValueError, match="too many rows"):
        rmi._call("rmi_kv_write", 2, FAKE, 1, 128 * 256, FAR, 0, 1 << 22, 128, 256, 1 << 22, None)
    p, a = rmi.RopeParams(1e6, 1.0, 0.0, 1.0, 1.0, 32.0, 1.0), rmi.RopeAxes((ctypes.c_int * 3)(32, 0, 0), 0)
    with pytest.raises(ValueError, match="attn_prep_axes"):
        rmi._call("rmi_attn_prep_axes", FAKE, 512, FAKE, FAKE, 1, FAKE, 1, ctypes.c_void_p(1 << 45), FAKE, None, FAKE, 1, 1, 128, 64,
                  ctypes.byref(p), ctypes.byref(a), 1e-6, 1 << 25, 1 << 26, None)
