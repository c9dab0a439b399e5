"""The pieces of the wide backward's products for a window (csrc/tc_bwd_wide.cuh, compiled here): a tile's contraction goes over the tiles that it
visits, once each, in pieces of bounded depth; dQ is stored only where one piece has all of it."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "z-transformer_b200", "csrc")
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include <random>
#include <vector>
#include "tc_bwd_wide.cuh"
using namespace zt;
int main() {
    std::mt19937 rng(5);
    const auto between = [&](int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); };
    int bad = 0, several = 0, stored = 0;
    for (int round = 0; round < 2000; ++round) {
        const int T = between(1, round % 8 ? 1500 : 6000), window = between(1, round % 3 ? T : 400), sinks = between(0, round % 4 ? 200 : T), Tp = (T + 127) / 128 * 128, nt = Tp / 128;
        tcw::WideParams p{};
        p.T = T, p.Tp = Tp, p.units = 2, p.n_heads = 2, p.n_kv_heads = 1, p.win = BwdWindow{window, sinks, 0};
        const tcw::WidePieces pieces = tcw::wide_pieces(p.win, Tp);
        p.pieces = pieces.n;
        p.in_turn = pieces.n == 1 && round % 2;
        // how often (product, head, tile) has been given each tile of its contraction, and by how many units
        std::vector<int> times((size_t)6 * nt * nt), units((size_t)6 * nt);
        for (int i = 0; i < 3 * nt * p.units * p.pieces; ++i) {
            const tcw::TriUnit w(p, i);
            if (w.n_steps <= 0) continue;
            if (w.n_steps * 64 > tcw::kPiece) ++bad;
            const size_t of = ((size_t)w.which * 2 + w.u) * nt + w.m0 / 128;
            ++units[of];
            for (int s = 0; s < w.n_steps; ++s) {
                const int k = w.contraction(s);
                if (k < 0 || k >= Tp) ++bad;
                else ++times[of * nt + k / 128];
            }
        }
        for (int which = 0; which < 3; ++which)
            for (int u = 0; u < 2; ++u)
                for (int m = 0; m < nt; ++m) {
                    const size_t of = ((size_t)which * 2 + u) * nt + m;
                    several += units[of] > 1, stored += which == 0 && pieces.dq == 1;
                    if (which == 0 && pieces.dq == 1 && units[of] != 1) ++bad;
                    for (int n = 0; n < nt; ++n) {
                        const int key = (which == 0 ? n : m) * 128, row = (which == 0 ? m : n) * 128;  // tiles
                        bool seen = false;  // by some row of some key, both inside the sequence
                        for (int t = row; t < row + 128 && !seen; ++t) seen = key <= t && (key + 127 > t - window || key < sinks);
                        if (times[of * nt + n] != (seen ? 2 : 0) && bad++ < 5)  // (steps of 64)
                            printf("T %d, window %d, %d sinks: product %d, tile %d, %d of %d\n", T, window, sinks, which, m, times[of * nt + n], n);
                    }
                }
    }
    printf("%d tiles of several units, %d stored, %d bad\n", several, stored, bad);
    return bad > 0 || several < 10000 || stored < 5000;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
def test_every_visited_tile_once(tmp_path):
    src = tmp_path / "pieces.cu"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "pieces")
    subprocess.check_call([NVCC, "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-o", exe, str(src), "-lcuda"])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
