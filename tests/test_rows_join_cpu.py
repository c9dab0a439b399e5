"""What the join of rows in parts reads (csrc/tc_rows.cuh, compiled here; without a device it takes a B200's 148 SMs): also of a row whose
weights are all NaN, nothing but the parts that were written."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "z-transformer_b200", "csrc")
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include "tc_rows.cuh"
using namespace zt;
int main() {
    int bad = 0, split = 0, partial = 0;
    const int heads[][3] = {{32, 8, 128}, {4, 2, 32}, {16, 16, 64}, {8, 2, 256}, {12, 4, 96}, {64, 1, 64}, {1, 1, 128}};
    for (const auto &h : heads)
        for (int batch : {1, 2, 5, 30})
            for (int rows : {1, 2, 9, 30, 77, 150, 280, 500, 900})
                for (int seen : {1, 200, 1000, 1008, 4096, 100000}) {
                    const int parts = tcr::row_parts(batch, rows, seen, h[0], h[1], h[2]);
                    if (parts < 2) continue;
                    ++split, partial += parts % 8 != 0;
                    const long long pairs = (long long)rows * h[0], written = parts * pairs * h[2];
                    for (const float weight : {0.f, 0.25f, NAN}) {
                        long long end = 0;  // of what the last row's last column is read from: eight parts at a time, as the kernel goes
                        for (int i0 = 0; i0 < parts; i0 += 8)
                            for (int i = 0; i < 8; ++i)
                                if (tcr::join_reads(i0 + i, parts, weight)) end = ((long long)(i0 + i) * pairs + pairs) * h[2];
                        if ((weight == 0.f ? end != 0 : end != written) && bad++ < 5)
                            printf("%d rows of %d sequences, %d keys, %d parts: weight %g reads up to %lld of %lld\n", rows, batch, seen, parts, weight, end, written);
                    }
                }
    printf("%d splits, %d of them no multiple of eight, %d bad\n", split, partial, bad);
    return bad > 0 || split < 100 || partial < 100;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
def test_a_row_of_nan_reads_the_parts_that_there_are(tmp_path):
    src = tmp_path / "join.cu"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "join")
    subprocess.check_call([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-o", exe, str(src), "-lcuda"])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
