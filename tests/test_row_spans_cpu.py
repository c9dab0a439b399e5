"""Which rows a tile of the attention over pages answers for (csrc/paged_kernels.cuh, compiled here), whatever the bounds are: every row between
the least and the greatest is one tile's, and a row is computed where it is one sequence's alone and no descent passes over it."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "z-transformer_b200", "csrc")
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#include "paged_kernels.cuh"
using namespace zt;
int main() {
    std::mt19937 rng(7);
    const auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
    long long bad = 0, descend = 0, computed = 0, shared = 0;
    for (int round = 0; round < 6000; ++round) {
        const int batch = 1 + upto(round % 3 == 0 ? 40 : 5), rows = 1 + upto(round % 2 ? 300 : 12), groups[] = {1, 2, 3, 4, 5, 16, 64, 300}, group = groups[upto(7)];
        std::vector<int> cu(batch + 1);
        for (int &c : cu) c = round % 5 == 0 ? upto(rows + 8) - 4 : upto(rows);
        if (round % 4 == 0) std::sort(cu.begin(), cu.end());
        if (round % 4 == 1) {  // ascending but for a place or two
            std::sort(cu.begin(), cu.end());
            std::swap(cu[upto(batch)], cu[upto(batch)]);
        }
        std::vector<int> c(batch + 1);
        for (int i = 0; i <= batch; ++i) c[i] = row_bound(cu.data(), rows, i);
        const bool ascend = std::is_sorted(c.begin(), c.end());
        descend += !ascend;
        const int low = *std::min_element(c.begin(), c.end()), high = *std::max_element(c.begin(), c.end());
        std::vector<int> tiles((size_t)rows * group), by(rows, -1);
        const long long slots = (long long)rows * group / 128 + batch;  // what is launched
        for (int slot = 0; slot < slots; ++slot) {
            const RowSpan s = row_span(cu.data(), batch, rows, group, slot);
            if (s.b < 0) continue;
            if (ascend && (s.begin != c[s.b] || s.end != c[s.b + 1] || std::min(s.upto, s.end) != s.end)) ++bad;
            const long long f0 = (slot - first_row_tile(s.begin, group, s.b)) * 128, flat = (long long)(s.end - s.begin) * group;
            for (long long f = f0; f < flat && f < f0 + 128; ++f) {
                const int row = s.begin + (int)(f / group);
                if (f < 0 || row >= rows) { ++bad; continue; }
                ++tiles[(size_t)row * group + f % group];
                if (row < s.upto) by[row] = s.b;
            }
        }
        for (int row = 0; row < rows; ++row) {
            const bool somebodys = low <= row && row < high;
            for (int h = 0; h < group; ++h) bad += tiles[(size_t)row * group + h] != (somebodys ? 1 : 0);
            int owners = 0, owner = -1, descents = 0;
            for (int b = 0; b < batch; ++b) {
                if (c[b] <= row && row < c[b + 1]) ++owners, owner = b;
                descents += c[b + 1] <= row && row < c[b];
            }
            shared += owners > 1;
            bad += by[row] != (owners == 1 && descents == 0 ? owner : -1);
            computed += by[row] >= 0;
        }
    }
    printf("%lld descending bounds, %lld rows computed, %lld in several bounds, %lld bad\n", descend, computed, shared, bad);
    return bad > 0 || descend < 2000 || computed < 10000 || shared < 10000;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
def test_every_row_is_one_tile_s(tmp_path):
    src = tmp_path / "spans.cu"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "spans")
    subprocess.check_call([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-o", exe, str(src), "-lcuda"])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
