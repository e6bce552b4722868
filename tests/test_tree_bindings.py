"""What the Python calls on quantised caches, drafted trees and logits check of their tensors before the library is entered (CPU:
stand-ins for tensors of a GPU, and a library that only notes its calls)."""
import pytest
import torch

import rapier_amd as rmi

F32, I32, I64, U8 = torch.float32, torch.int32, torch.int64, torch.uint8


class Tensor:
    def __init__(self, dtype, device=0, numel=1 << 20, at=1 << 20):
        self.dtype, self.device, self.size, self.at = dtype, device, numel, at

    def get_device(self):
        return self.device

    def data_ptr(self):
        return self.at if self.size else 0

    def numel(self):
        return self.size


class Stream:
    def __init__(self, device):
        self.device_index, self.cuda_stream = device, 77


def kv_write(t, **kw):
    rmi.kv_write(rmi.KV_I8, t["src"], 1024, t["cache"], 0, kw.pop("n", 3), 4, 256, 100, **kw)


def kv_read(t, **kw):
    rmi.kv_read(rmi.KV_I8, t["cache"], t["out"], 1024, 0, kw.pop("n", 3), 4, 256, 100, **kw)


def kv_compact(t, **kw):
    rmi.kv_compact(rmi.KV_I8, [t["first"], t["second"]], t["pos"], t["path"], t["count"], 4, 4, 256, 100, **kw)


def prep(t, **kw):
    rmi.attn_prep_axes(t["q3"], 10240, t["qn"], t["kn"], 1, t["k"], 1, t["v"], t["pos"], t["axis_pos"], t["qout"], 16, 4, 256, 64, 1e6, 1.0,
                       0.0, (12, 10, 10), True, 1e-6, 1, 100, **kw)


def tree(t, **kw):
    rmi.gqa_tree_decode(t["q"], 1, t["k"], 1, t["v"], t["pos"], t["masks"], t["gate"], 10240, t["y"], 4096, t["q8"], 4608, t["workspace"], 16, 4,
                        256, 1, 100, 1, 0.06, **kw)


def logits(t, **kw):
    rmi.logits_process(t["logits"], 1000, 1, 1000, t["out"], 1000, t["history"], t["history_len"], 9, 0, t["draft"], t["masks"], 1, 1.5, 0.5,
                       0.25, t["bias_ids"], t["bias_vals"], 3, t["allow"], 32, **kw)


# every tensor argument and its type
CALLS = {
    kv_write: {"src": F32, "cache": U8},
    kv_read: {"cache": U8, "out": torch.float16},
    kv_compact: {"first": U8, "second": U8, "pos": I32, "path": I32, "count": I32},
    prep: {"q3": F32, "qn": F32, "kn": F32, "k": U8, "v": U8, "pos": I32, "axis_pos": I32, "qout": F32},
    tree: {"q": F32, "k": U8, "v": U8, "pos": I32, "masks": I64, "gate": F32, "y": F32, "q8": U8, "workspace": U8},
    logits: {"logits": F32, "out": F32, "history": I32, "history_len": I32, "draft": I32, "masks": I64, "bias_ids": I32, "bias_vals": F32,
             "allow": I32},
}
EACH = [pytest.param(f, name, id=f"{f.__name__}-{name}") for f, ts in CALLS.items() for name in ts]


@pytest.fixture
def entered(monkeypatch):
    calls = []
    monkeypatch.setattr(rmi, "_call", lambda *a: calls.append(a))
    monkeypatch.setattr(rmi, "_gpu", (lambda: 0, lambda at: 55))
    return calls


def tensors(f):
    return {name: Tensor(dtype) for name, dtype in CALLS[f].items()}


@pytest.mark.parametrize("f", list(CALLS), ids=lambda f: f.__name__)
def test_tensors_of_the_current_gpu_reach_the_library(entered, f):
    f(tensors(f))
    f(tensors(f), stream=5)
    f(tensors(f), stream=Stream(0))
    assert [c[-1] for c in entered] == [55, 5, 77]


@pytest.mark.parametrize("where", [-1, 1])
@pytest.mark.parametrize("f,name", EACH)
def test_each_tensor_has_to_be_on_the_current_gpu(entered, f, name, where):
    t = tensors(f)
    t[name].device = where
    for kw in ({}, {"stream": 5}):
        with pytest.raises(ValueError, match="not on the current GPU"):
            f(t, **kw)
    assert not entered


@pytest.mark.parametrize("f", list(CALLS), ids=lambda f: f.__name__)
def test_another_gpu_than_the_current_one(entered, f):
    t = tensors(f)
    for x in t.values():
        x.device = 1
    with pytest.raises(ValueError, match="not on the current GPU"):
        f(t)
    with pytest.raises(ValueError, match="stream"):
        f(tensors(f), stream=Stream(1))
    assert not entered


@pytest.mark.parametrize("f,name", [p for p in EACH if p.values[0] not in (kv_write, kv_read) and CALLS[p.values[0]][p.values[1]] is not U8])
def test_each_tensor_has_to_be_of_its_type(entered, f, name):
    """a narrower tensor would be read or written past its end"""
    t = tensors(f)
    right = t[name].dtype
    for wrong in {F32, I32, I64, torch.float16, torch.bfloat16, torch.float64, torch.int16, torch.int8, torch.bool} - {right}:
        t[name].dtype = wrong
        with pytest.raises(ValueError, match="where the library takes"):
            f(t)
    assert not entered
    for same in {F32: (U8,), I32: (torch.uint32, U8), I64: (torch.uint64, U8)}[right]:   # U8: raw memory
        t[name].dtype = same
        f(t)


@pytest.mark.parametrize("f,name", [(kv_write, "cache"), (kv_read, "cache"), (kv_compact, "second"), (prep, "k"), (tree, "v"), (tree, "workspace")])
def test_caches_and_workspaces_are_memory_of_any_type(entered, f, name):
    for dtype in (torch.float16, torch.int16, F32, I64):
        t = tensors(f)
        t[name].dtype = dtype
        f(t)
    assert len(entered) == 4


@pytest.mark.parametrize("call,name", [(rmi.kv_write, "src"), (rmi.kv_read, "out")], ids=["kv_write", "kv_read"])
@pytest.mark.parametrize("dtype", [F32, torch.float16])
def test_no_rows_of_an_empty_tensor(monkeypatch, call, name, dtype):
    """torch's empty tensors have no address; through the library itself, which launches nothing for no rows"""
    monkeypatch.setattr(rmi, "_gpu", (lambda: 0, lambda at: 55))
    rows, cache = Tensor(dtype, numel=0), Tensor(U8)
    args = (rows, 1024, cache) if name == "src" else (cache, rows, 1024)
    for first in (0, 100):
        call(rmi.KV_I8, *args, first, 0, 4, 256, 100)
    with pytest.raises(ValueError, match="invalid"):
        call(rmi.KV_I8, *args, 0, 1, 4, 256, 100)
    with pytest.raises(ValueError, match="invalid"):
        call(rmi.KV_I8, *args, 101, 0, 4, 256, 100)


def test_rotary_values_that_change_in_place(entered):
    """elements of tensors as base, factor and sections: every call has what they hold at that call"""
    base, factor, sections = torch.tensor(1e4), torch.tensor(2.0), torch.tensor([12, 10, 10])
    views = [sections[i] for i in range(3)]
    t = tensors(prep)
    for new in ((1e4, 2.0, (12, 10, 10)), (1e6, 4.0, (10, 11, 11)), (5e5, 8.0, (32, 0, 0))):
        base.fill_(new[0])
        factor.fill_(new[1])
        sections.copy_(torch.tensor(new[2]))
        rmi.attn_prep_axes(t["q3"], 10240, t["qn"], t["kn"], 1, t["k"], 1, t["v"], t["pos"], t["axis_pos"], t["qout"], 16, 4, 256, 64, base,
                           factor, 32768.0, views, False, 1e-6, 1, 100)
        blocks = [a._obj for a in entered[-1] if hasattr(a, "_obj")]
        assert (blocks[0].freq_base, blocks[0].factor) == new[:2]
        assert tuple(blocks[1].section) == new[2]
    with pytest.raises(TypeError):
        rmi.attn_prep_axes(t["q3"], 10240, t["qn"], t["kn"], 1, t["k"], 1, t["v"], t["pos"], t["axis_pos"], t["qout"], 16, 4, 256, 64, 1e4,
                           1.0, 0.0, (12.5, 9.5, 10.0), False, 1e-6, 1, 100)
