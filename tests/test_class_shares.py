"""The shares of a row's classes (csrc/class_shares.h), compiled for the host: the parts that they read of each component are the component, up to the
largest rows that the distillation takes."""
import os
import re
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "phoenix_core_b200", "csrc")
SOURCE = r"""
#include "class_shares.h"
#include <algorithm>
#include <cstdio>
int main() {
    const int rows[][2] = {{1, 1}, {1, 50001}, {4, 250}, {8, 10654}, {1, 1 << 30}, {1, (1 << 30) + 1}, {1, 1200000000}, {1, 2147483647}, {2, 1073741823}, {4, 500000000},
                           {8, (1 << 28) - 8}, {8, (1 << 28) - 1}};
    for (const auto& r : rows) {
        const int comps = r[0], units = r[1], classes = comps * units;
        for (int shares = 1; shares <= 8; shares *= 2) {
            if (classes < shares) continue;
            int next = 0;                                      // classes are visited in order, each once
            for (int s = 0; s < shares; ++s) {
                const int lo = pcb::share_start(classes, s, shares), hi = pcb::share_start(classes, s + 1, shares);
                for (int c = lo / units, end = pcb::components_below(hi, units); c < end; ++c) {
                    const int a = std::max(lo, c * units), b = std::min(hi, (c + 1) * units);
                    if (c >= comps || a != next || b <= a) { std::printf("%d x %d, share %d of %d: [%d, %d) behind %d\n", comps, units, s, shares, a, b, next); return 1; }
                    next = b;
                }
            }
            if (next != classes) { std::printf("%d x %d in %d shares: %d classes visited\n", comps, units, shares, next); return 1; }
        }
    }
    return 0;
}
"""


def test_every_class_once(tmp_path):
    source, program = tmp_path / "shares.cpp", tmp_path / "shares"
    source.write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-I" + CSRC, "-o", str(program), str(source)])
    result = subprocess.run([str(program)], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout


def test_the_kernels_take_these():
    text = open(os.path.join(CSRC, "distill.cu")).read()
    assert len(re.findall(r"share_start\(classes, split, p\.splits\), hi = share_start\(classes, split \+ 1, p\.splits\)", text)) == 2
    assert len(re.findall(r"components_below\(hi, p\.units\)", text)) == 1 and "p.units - 1)" not in text
