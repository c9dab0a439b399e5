"""Bounds of new rows that do not ascend, so that sequences claim the same rows: what the append writes is what it counts, and the attention
computes the rows that are one sequence's alone and makes the others NaN."""
import pytest
import torch
from test_gpu_paged import Case, near, rand

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


@pytest.mark.parametrize("bounds,rows", BOUNDS + [([0, 300, 250, 260, 310], 310), ([20, 10, 200, 150, 400, 380, 420], 430), ([0, 150, 149, 300], 300)])
@pytest.mark.parametrize("H,G,D,window", [(8, 2, 64, 0), (4, 1, 128, 40), (8, 2, 256, 0), (32, 8, 128, 0)])
def test_attention_computes_the_rows_of_one_sequence(zt, bounds, rows, H, G, D, window):
    B, page = len(bounds) - 1, 16
    own = [hi - lo if 0 <= lo <= hi <= rows else 0 for lo, hi in zip(bounds, bounds[1:])]
    past = [(37 * b) % 150 for b in range(B)]
    c = Case(own, past, H, G, D, page, window, 2 if window else 0, seed=rows)
    c.N, c.q, c.cu = rows, rand(rows, H * D, seed=5), torch.tensor(bounds, dtype=torch.int32, device="cuda")
    ws = zt.PagedWorkspace(B, rows, c.table.shape[1] * page, H, G, D)
    ws.buf.fill_(255)
    given = torch.full_like(c.q, 9.0)
    out, lse = c.call(zt, workspace=ws, out=given)
    again, _ = c.call(zt, workspace=ws, out=torch.full_like(c.q, 9.0))
    assert torch.equal(out.nan_to_num(7.0), again.nan_to_num(7.0))  # whoever comes first
    clip = [min(max(x, 0), rows) for x in bounds]
    for row in range(rows):
        owners = [b for b in range(B) if clip[b] <= row < clip[b + 1]]
        down = any(clip[b + 1] <= row < clip[b] for b in range(B))
        if not min(clip) <= row < max(clip):
            assert (out[row] == 9.0).all(), row
        elif len(owners) == 1 and not down and own[owners[0]]:
            continue
        else:
            assert out[row].isnan().all() and lse[row].isnan().all(), row
    computed = 0
    for b in range(B):
        lo, hi = max(clip[:b + 1]), min(clip[b + 1:])
        if own[b] and lo < hi:
            ref, ref_lse = c.reference(b)
            at = slice(lo - bounds[b], hi - bounds[b])
            near(out[lo:hi], ref[at], b)
            near(lse[lo:hi], ref_lse[at], b)
            computed += hi - lo
    assert computed == int((~lse.isnan().any(1) & (out != 9.0).all(1)).sum())
    assert ws.bad_sequences() == sum(not 0 <= lo <= hi <= rows for lo, hi in zip(bounds, bounds[1:])) and zt.lib.tc_status() == 0
