"""The blocks of a window's backward (csrc/tc_split.cuh, compiled here): every query tile that some key of a key tile is seen from is walked once
for it, key tiles of several blocks add, and what a launch has along x stays within its limit for numbers that the calls admit."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "z-transformer_b200", "csrc")
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include <cstdio>
#include <random>
#include <vector>
#include "zt_common.cuh"
#include "tc_split.cuh"
using namespace zt;
int main() {
    std::mt19937 rng(3);
    long long bad = 0, adding = 0;
    const auto between = [&](int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); };
    for (int round = 0; round < 3000; ++round) {
        const int rows = round % 2 ? 64 : 128, T = between(1, round % 10 == 0 ? 20000 : 1500), window = between(1, round % 3 ? T : 200), sinks = between(0, round % 4 ? 300 : T);
        const BwdWindow w{window, sinks, (window + 127) / rows + 2};
        const int kts = (T + 127) / 128, qts = (T + rows - 1) / rows;
        const long long blocks = window_grid(w, T, rows, 1);
        bad += window_grid(w, T, rows, 5) != 5 * blocks;
        std::vector<unsigned char> walked((size_t)kts * qts);
        std::vector<int> of_tile(kts), adds(kts);
        for (int i = 0; i < blocks; ++i) {
            const WindowBlock x = window_block(w, T, i, rows);
            if (x.kt < 0 || x.kt >= kts || x.qi0 < 0 || x.n_q > qts || x.qi0 >= x.n_q) { ++bad; continue; }
            ++of_tile[x.kt], adds[x.kt] += x.adds;
            for (int q = x.qi0; q < x.n_q; ++q) ++walked[(size_t)x.kt * qts + q];
        }
        for (int kt = 0; kt < kts; ++kt) {
            bad += adds[kt] != (of_tile[kt] > 1 ? of_tile[kt] : 0);  // all of them, or the only one does not
            adding += of_tile[kt] > 1;
            for (int q = 0; q < qts; ++q) {
                // the tile's last key from the tile's last query on, or its first key, where it is a sink, from any query at or behind it
                const int k0 = kt * 128, k1 = k0 + 127 < T ? k0 + 127 : T - 1, t0 = q * rows, t1 = t0 + rows - 1 < T ? t0 + rows - 1 : T - 1;
                bool seen = false;
                if (t1 >= k0) seen = k1 > t0 - window || k0 < sinks;
                const int n = walked[(size_t)kt * qts + q];
                bad += n > 1 || (seen && n == 0);
            }
        }
    }
    // beyond what y takes, within what x takes
    const int big[][5] = {{131072, 64, 32768, 64, 8}, {65536, 1, 65535, 64, 64}, {131072, 256, 65536, 64, 8}, {131072, 64, 32768, 128, 128}};
    for (const auto &b : big) {
        const BwdWindow w{b[1], b[2], (b[1] + 127) / b[3] + 2};
        const long long n = window_grid(w, b[0], b[3], b[4]);
        if (n <= 65535 || n > 0x7fffffffll) ++bad, printf("T %d, window %d, %d sinks: %lld blocks\n", b[0], b[1], b[2], n);
    }
    printf("%lld key tiles of several blocks, %lld bad\n", adding, bad);
    return bad > 0 || adding < 1000;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
def test_every_visit_once(tmp_path):
    src = tmp_path / "blocks.cu"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "blocks")
    subprocess.check_call([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-o", exe, str(src), "-lcuda"])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_a_window_s_launch_has_its_blocks_along_x():
    """Where a grid has 2^31 - 1 of them; along y it has 65535."""
    for f in ("tc_bwd_fused.cuh", "tc_bwd_fused64.cuh"):
        text = open(os.path.join(CSRC, f)).read()
        assert "const dim3 grid = win ? dim3((unsigned)window_grid(" in text and "window_block(p.win, p.T, (int)blockIdx.y" not in text, f
