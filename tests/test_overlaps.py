"""Calls whose outputs lie on their inputs are refused before any device work (CPU); the test of strided rows itself against
all bytes, in a small program."""
import ctypes
import os
import shutil
import subprocess
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = textwrap.dedent(r"""
    #include "overlap.h"
    #include <cstdio>
    #include <set>
    #include <random>
    int main() {
        std::mt19937 rng(1);
        auto draw = [&](int lo, int hi) { return lo + static_cast<int>(rng() % (hi - lo + 1)); };
        int shared = 0;
        for (int i = 0; i < 200000; ++i) {
            rmi::RowSet s[2];
            std::set<long long> bytes[2];
            for (int k = 0; k < 2; ++k) {
                long long p = 1000 + draw(0, 60);
                s[k] = {reinterpret_cast<const void*>(p), draw(1, 7), draw(-25, 25), draw(1, 12)};
                for (long long r = 0; r < s[k].n; ++r)
                    for (long long b = 0; b < s[k].bytes; ++b) bytes[k].insert(p + r * s[k].stride + b);
            }
            bool want = false;
            for (long long b : bytes[0]) want = want || bytes[1].count(b);
            shared += want;
            if (rmi::rows_overlap(s[0], s[1]) != want) {
                for (auto& x : s) std::printf("%p %lld %lld %lld\n", x.p, x.n, x.stride, x.bytes);
                return 1;
            }
        }
        std::printf("%d\n", shared);
        return shared > 50000 && shared < 190000 ? 0 : 2;
    }
""")


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_strided_rows_against_all_bytes(tmp_path):
    src, exe = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "rapier_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.fixture(scope="module")
def rmi():
    import rapier_amd
    rapier_amd.lib()
    return rapier_amd


BASE = 1 << 30


def at(offset):
    return ctypes.c_void_p(BASE + offset)


# a cache of 100 positions x 4 heads x 256 at BASE, positions 10 .. 14; rows outside: five of 4 KB (fp32) or 2 KB
@pytest.mark.parametrize("name", ["rmi_kv_write", "rmi_kv_read"])
@pytest.mark.parametrize("type_,rows,f16,stride", [
    (0, 10 * 2048, 1, 1024), (0, 15 * 2048 - 4, 0, 1024), (0, 10 * 2048 - 5 * 2048 + 2, 1, 1024), (0, 10 * 2048 - 4096 - 8192 * 2 + 4, 0, 2048),
    (1, 10 * 256, 0, 1024), (1, (2 * 100 + 14) * 256 + 252, 0, 1024), (1, 4 * 100 * 256 + (3 * 100 + 14) * 8 + 4, 0, 1024),
    (1, 4 * 100 * 256 + 10 * 8 - 5 * 2048 + 2, 1, 1024), (2, (100 + 10) * 128, 1, 1024), (2, 4 * 100 * 128 + (100 + 12) * 8, 1, 1024)])
def test_rows_on_their_own_cache_rows(rmi, name, type_, rows, f16, stride):
    a = (at(rows), f16, stride, at(0)) if name == "rmi_kv_write" else (at(0), at(rows), f16, stride)
    with pytest.raises(ValueError, match="lies on"):
        rmi._call(name, type_, *a, 10, 5, 4, 256, 100, None)


# caches whose rows and bytes pass 32 bits: 2^26 positions x 64 heads x 256, the last five of them
FIRST = (1 << 26) - 5
HUGE = {0: [64 * FIRST * 512, 64 * FIRST * 512 + 5 * 64 * 512 - 4],
        1: [FIRST * 256, 63 * (1 << 26) * 256 + FIRST * 256 + 1000, 64 * (1 << 26) * 256 + FIRST * 8, 64 * (1 << 26) * (256 + 8) - 4],
        2: [FIRST * 128, 64 * (1 << 26) * 128 + (31 * (1 << 26) + FIRST) * 8]}


@pytest.mark.parametrize("name", ["rmi_kv_write", "rmi_kv_read"])
@pytest.mark.parametrize("type_,rows", [(t, r) for t in HUGE for r in HUGE[t]])
def test_rows_on_their_own_rows_of_a_huge_cache(rmi, name, type_, rows):
    a = (at(rows), 0, 64 * 256, at(0)) if name == "rmi_kv_write" else (at(0), at(rows), 0, 64 * 256)
    with pytest.raises(ValueError, match="lies on"):
        rmi._call(name, type_, *a, FIRST, 5, 64, 256, 1 << 26, None)


@pytest.mark.parametrize("out,ncols,col_stride,out_stride", [
    (4, 1, 1000, 1000), (-4, 1, 1000, 1000), (3996, 1, 1000, 1000), (4000, 2, 1000, 1000), (-4 * 1004, 3, 1004, 1004), (4, 64, 1000, 1000),
    (3996, 2, 2000, 2000), (4 * 2000, 3, 2000, 1000), (4 * 63 * 2000 + 4 * 999, 64, 2000, 2000), (-4 * 63 * 3001 + 400, 64, 2000, 3001)])
def test_logits_on_other_logits(rmi, out, ncols, col_stride, out_stride):
    p = rmi.Penalties(1.0, 0.0, 0.0, 0)
    with pytest.raises(ValueError, match="lies on"):
        rmi._call("rmi_logits_process", at(0), 1000, ncols, col_stride, at(out), out_stride, None, None, 0, None, None, 0, ctypes.byref(p), None,
                  None, 0, None, 0, None)


# 16 heads on 4 KV heads of 256, 8 tokens: q 128 KB, y the same, q8 36 KB, caches of 1000 positions, 1 MB each as I8
TREE = {"q": 0, "k": 1 << 24, "v": 1 << 25, "gate": 1 << 26, "y": 1 << 20, "q8": 1 << 21, "ws": 1 << 27}


@pytest.mark.parametrize("moved,to,extra", [
    ("y", 16, {}), ("y", (1 << 17) - 4, {}), ("y", 0, {"ys": 4100}), ("y", -4 * 4096, {"ys": 4100}), ("y", (1 << 24) + 64, {}), ("y", (1 << 25) - 64, {}),
    ("y", 1 << 26, {}), ("y", (1 << 26) + 4 * 256, {"ys": 10240}), ("y", (1 << 26) + 4 * 8188, {"ys": 10240}), ("y", (1 << 27) + 400000, {}),
    ("y", (1 << 21) + 8 * 4608 - 4, {}), ("q8", 0, {}), ("q8", (1 << 24) + 1000000, {}), ("q8", (1 << 26) + 4 * 10240 * 7 + 4 * 256, {}),
    ("ws", 1 << 16, {}), ("ws", (1 << 24) + 4096, {}), ("ws", (1 << 25) - 4096, {}), ("ws", 1 << 20, {}), ("ws", (1 << 21) - 16, {}),
    ("ws", (1 << 26) + 4096, {})])
def test_tree_outputs_on_inputs(rmi, moved, to, extra):
    p = {k: at(v) for k, v in {**TREE, moved: to}.items()}
    with pytest.raises(ValueError, match="lies on"):
        rmi._call("rmi_gqa_tree_decode", p["q"], 1, p["k"], 1, p["v"], at(1 << 28), None, p["gate"], 10240, p["y"], extra.get("ys", 4096), p["q8"], 4608,
                  p["ws"], 16, 4, 256, 8, 1000, 1, 0.0625, None)


@pytest.mark.parametrize("qout,k,v", [(0, 1 << 24, 1 << 25), (4 * 10240 * 5 - 4, 1 << 24, 1 << 25), (-4 * 4096 * 5 + 4, 1 << 24, 1 << 25),
                                      (4 * 256, 1 << 24, 1 << 25), ((1 << 24) + 64, 1 << 24, 1 << 25), ((1 << 25) - 64, 1 << 24, 1 << 25),
                                      (1 << 26, 4 * 10240 * 4, 1 << 25), (1 << 26, 1 << 24, -1024), (1 << 26, 1 << 24, (1 << 24) + 4096)])
def test_prep_outputs_on_inputs(rmi, qout, k, v):
    """five tokens of 16 + 4 heads of 256, I8 caches of 100 positions"""
    p, a = rmi.RopeParams(1e6, 1.0, 0.0, 1.0, 1.0, 32.0, 1.0), rmi.RopeAxes((ctypes.c_int * 3)(32, 0, 0), 0)
    with pytest.raises(ValueError, match="lies on|overlap"):
        rmi._call("rmi_attn_prep_axes", at(0), 10240, at(1 << 28), at(1 << 28), 1, at(k), 1, at(v), at(1 << 28), None, at(qout), 16, 4, 256, 64,
                  ctypes.byref(p), ctypes.byref(a), 1e-6, 5, 100, None)
