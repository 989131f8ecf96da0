"""The address and work arithmetic that the paged-cache kernels share (csrc/kv_addr.h), compiled for the CPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = r"""
#include "kv_addr.h"
#include <stdio.h>
int main() {
    // two pages of 16 positions named, one id too large, one negative
    const int32_t row[4] = {3, 7, 8, -1};
    const int64_t pos[] = {0, 15, 16, 31, 32, 48, 63, 64, 1LL << 40, -1};
    const int32_t want[] = {3, 3, 7, 7, -1, -1, -1, -1, -1, -1};
    for (int i = 0; i < 10; ++i)
        if (kv_page_of(row, 64, 4, 8, pos[i]) != want[i]) return printf("page of %lld\n", (long long)pos[i]), 1;
    if (kv_page_or_none(2147483647, 2147483647) != -1 || kv_page_or_none(-2147483647, 5) != -1) return printf("ids\n"), 1;
    // every tile belongs to one wavefront, every wavefront has one tile at least, runs differ by one tile at most
    for (int64_t W = 1; W <= 70; ++W)
        for (int64_t T = W; T <= 300; ++T) {
            if (kv_first_tile(0, T, W) != 0 || kv_first_tile(W, T, W) != T) return printf("ends\n"), 1;
            for (int64_t w = 0; w < W; ++w) {
                const int64_t a = kv_first_tile(w, T, W), b = kv_first_tile(w + 1, T, W);
                if (b - a < T / W || b - a > T / W + 1) return printf("run %lld %lld\n", (long long)T, (long long)W), 1;
                for (int64_t t = a; t < b; ++t)
                    if (kv_wave_of_tile(t, T, W) != w) return printf("tile %lld\n", (long long)t), 1;
            }
        }
    const int64_t T = 1LL << 40, W = 2048;
    for (int64_t w = 0; w < W; ++w)
        if (kv_wave_of_tile(kv_first_tile(w, T, W), T, W) != w) return printf("far\n"), 1;
    return 0;
}
"""


def test_addresses_and_runs(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    c = tmp_path / "t.cpp"
    c.write_text(SRC)
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(HERE, "..", "vortex_amd", "csrc"), str(c), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
