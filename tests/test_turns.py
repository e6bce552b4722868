"""cos and sin of an angle in turns (rapier_amd/csrc/turns.h), compiled for the CPU, against long double."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rapier_amd", "csrc")

# the largest errors over [-1/8, 1/8] of a turn, then over [-1/2, 1/2] (what is left of an angle by its whole turns)
PROGRAM = r"""
#define __host__
#define __device__
#define __forceinline__ inline
#include "turns.h"
#include <cmath>
#include <cstdio>
int main() {
    const long double tau = 6.283185307179586476925286766559005768L;
    for (int part = 8; part >= 2; part -= 6) {
        const int n = 1 << 21;
        long double off = 0.0L;
        for (int i = -n; i <= n; ++i) {
            const double t = static_cast<double>(i) / n / part;
            double c, s;
            rmi::cos_sin_turns(t, &c, &s);
            off = std::fmax(off, std::fmax(std::fabs(c - std::cos(tau * t)), std::fabs(s - std::sin(tau * t))));
        }
        std::printf("%.4Le\n", off);
    }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
@pytest.mark.parametrize("contract", ["off", "fast"])   # the GPU's compiler fuses a product and a sum where it can
def test_turns_within_their_bound(tmp_path, contract):
    """x is off by at most 1.5 units of 2^-53 (2 pi as stored, the product) times pi / 4, of which cos and sin take sqrt(1/2) at most
    where it is that large, 0.9e-16; x^2 times the inner sum (|.| < 0.31) carries 3 units, 1.0e-16; the last sum half a unit of 1,
    1.1e-16; the terms left out 0.5e-16: 3.5e-16 in all, within 2^-51 = 4.4e-16"""
    if contract == "fast" and " fma " not in open("/proc/cpuinfo").read():
        pytest.skip("no fused multiply-add on this CPU")
    src, exe = tmp_path / "turns.cpp", tmp_path / "turns"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", f"-ffp-contract={contract}", *(["-mfma"] if contract == "fast" else []), "-I", CSRC, str(src), "-o",
                    str(exe)], check=True)
    off = [float(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert len(off) == 2 and max(off) <= 2.0 ** -51, off
