"""Where min-p ends (csrc/hq4_min_p.cuh), compiled for the host: the value is the
smallest one that stays, found in a bounded number of steps whatever the
temperature, the maximum and min_p are."""
import os
import shutil
import subprocess

import pytest

from hetero_infer_b200 import build

SOURCE = r"""
#include <cstdio>
#include "hq4_min_p.cuh"
using namespace hq4;
int main() {
    const float inf = INFINITY, tops[] = {0.0f, 10.0f, 20.0f, -20.0f, 1e-3f, 1e-40f, -1e-40f, 1e30f, -1e30f, FLT_MAX, -FLT_MAX, 65504.0f,
                                          1000.0f, 88.722839f, -0.5f};
    const float temps[] = {1.0f, 0.7f, 1e-7f, 1e-45f, 1e-38f, 1e9f, 1e30f, FLT_MAX, inf, 2.0f};
    const float mins[] = {1.0f, 7.0f, inf, 0.5f, 0.1f, 1e-9f, 2.0611537e-9f, 1e-38f, 1e-45f, 0.99999994f, 1e-30f};
    int most_calls = 0, wrong = 0, n = 0;
    for (float top : tops)
        for (float t : temps)
            for (int i = 0; i < 11 + 40; i++) {
                const double oct = 1.4426950408889634074 / (double)t;
                // after the fixed ones: the border at 0, where the floats are densest, and a few roundings beside it
                const float m = i < 11 ? mins[i] : (float)exp2(-(double)top * oct * (1.0 + (i - 31) * 0x1p-53));
                if (!(m > 0.0f)) continue;
                n++;
                const float end = min_p_end(m, top, oct);
                if (!(oct > 0.0)) {
                    wrong += end != -FLT_MAX;
                    continue;
                }
                const double most = -log2((double)fminf(m, 1.0f));
                int calls = 0;
                auto stays = [&](uint32_t k) {
                    calls++;
                    return ((double)top - (double)order_value(k)) * oct <= most;
                };
                const uint32_t lowest = order_bits(-FLT_MAX), last = order_bits(top);
                const float guess = (float)fmax((double)top - most / oct, -(double)FLT_MAX);
                const uint32_t k = first_that_stays(lowest, order_bits(fminf(guess, top)), last, stays);
                most_calls = calls > most_calls ? calls : most_calls;
                if (!(order_value(k) == end) || k < lowest || k > last || !stays(k) || (k > lowest && stays(k - 1))) {
                    wrong++;
                    printf("top %g temperature %g min_p %g: %g\n", top, t, m, end);
                }
                // any guess gives the same
                for (uint32_t g : {lowest, last, lowest + (last - lowest) / 3})
                    wrong += first_that_stays(lowest, g, last, stays) != k;
            }
    printf("%d %d %d\n", n, wrong, most_calls);
    return 0;
}
"""


def test_min_p_end(tmp_path):
    if not (os.path.exists(build.nvcc()) or shutil.which(build.nvcc())):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "min_p.cu", tmp_path / "min_p"
    src.write_text(SOURCE)
    subprocess.run([build.nvcc(), "-std=c++17", "-O2", *build.ARCH_FLAGS, f"-I{build.CSRC}", str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout
    n, wrong, most_calls = map(int, out.split("\n")[-2].split())
    assert n > 3000 and wrong == 0, out
    assert most_calls <= 34
