"""Bounds of new rows that do not ascend, so that sequences claim the same rows: what the append writes is what it counts."""
import pytest
import torch
from test_gpu_paged import rand

pytestmark = pytest.mark.gpu

#: bounds, rows: a row of two sequences, of four, of sequences with another's rows inside; bounds out of range among them
BOUNDS = [
    ([0, 5, 3, 8], 8), ([0, 2, 1], 3), ([0, 9, 2, 9, 4, 9, 1, 9], 9), ([0, 40, 30, 33, 60], 60), ([5, 0, 3], 5), ([0, 4, -1, 6, 12], 10), ([7, 3, 0], 7),
    ([0, 3, 6, 9], 9), ([2, 2, 4, 4, 7], 9),
]


@pytest.mark.parametrize("bounds,rows", BOUNDS)
@pytest.mark.parametrize("width", [32, 2048])
def test_append_writes_what_it_counts(zt, bounds, rows, width):
    page, B, slots = 4, len(bounds) - 1, 20
    table = torch.randperm(B * slots).int().view(B, slots)
    kn, vn = rand(rows, width, seed=1), rand(rows, width, seed=2)
    kp, vp = rand(B * slots, page, width, seed=3), rand(B * slots, page, width, seed=4)
    filled = [(5 * b) % 7 for b in range(B)]
    n, skipped = torch.tensor(filled, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    want_k, want_v, counts, bad = kp.clone(), vp.clone(), list(filled), 0
    for b, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo < 0 or hi < lo or hi > rows:
            bad += 1
            continue
        for i in range(lo, hi):
            s = filled[b] + i - lo
            want_k[table[b, s // page], s % page], want_v[table[b, s // page], s % page] = kn[i], vn[i]
        counts[b] += hi - lo
    zt.paged_append(kp, vp, table.cuda(), n, kn, vn, cu_rows=torch.tensor(bounds, dtype=torch.int32, device="cuda"), skipped=skipped)
    assert n.tolist() == counts and int(skipped) == bad
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
