"""The backward norms' grids beside an SM margin (csrc/sm_share.h), compiled for the host."""
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "phoenix_core_b200", "csrc")
SOURCE = r"""
#include "sm_share.h"
#include <cstdio>
int main() {
    for (int sms = 2; sms <= 160; ++sms)
        for (int places = 1; places <= 8; places *= 2)
            for (int ctas = 1; ctas <= 320; ++ctas) {
                const int got = pcb::ctas_beside(ctas, places, sms);
                const int least = ctas < places ? ctas : places;      // a CTA for each place that rows start at, where there are rows
                const bool fits = got <= sms || got == least;
                if (got < least || got > ctas || !fits || (ctas <= sms && got != ctas) || (ctas > sms && ctas > places && got % places != 0)) {
                    std::printf("%d CTAs, %d places, %d SMs: %d\n", ctas, places, sms, got);
                    return 1;
                }
            }
    return 0;
}
"""


def test_ctas_beside_a_margin(tmp_path):
    source, program = tmp_path / "share.cpp", tmp_path / "share"
    source.write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-I" + CSRC, "-o", str(program), str(source)])
    result = subprocess.run([str(program)], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout
