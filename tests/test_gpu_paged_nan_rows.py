"""Rows over pages that come out as NaN where the keys are split into parts: the join of the parts stays inside the workspace, which ends
in front of other tensors, and the rows beside them are right."""
import math

import pytest
import torch
from test_gpu_paged import Case, near

pytestmark = pytest.mark.gpu
GUARD = 64 << 20


def inside(zt, c, page):
    """A workspace of the least size, cut from a larger allocation; returns it and what lies behind it."""
    ws = zt.PagedWorkspace(len(c.rows), c.N, c.table.shape[1] * page, c.H, c.G, c.D)
    whole = torch.full((ws.nbytes + GUARD,), 255, dtype=torch.uint8, device="cuda")
    ws.buf = whole[:ws.nbytes]
    return ws, whole[ws.nbytes:]


@pytest.mark.parametrize("rows,past,H,G,D,page", [
    ([77], [931], 32, 8, 128, 16), ([280], [720], 32, 8, 128, 8), ([90, 30], [600, 900], 16, 4, 64, 16), ([200], [1500], 16, 4, 256, 16),
    ([30], [600], 16, 4, 256, 16), ([17], [2000], 32, 8, 128, 64),
])
@pytest.mark.parametrize("what", ["counts", "page", "q"])
def test_rows_of_nan_in_parts(zt, rows, past, H, G, D, page, what):
    c = Case(rows, past, H, G, D, page, seed=31)
    ws, behind = inside(zt, c, page)
    last = rows[-1]
    nan = torch.zeros(c.N, H, dtype=torch.bool, device="cuda")
    if what == "counts":
        c.n_keys[-1] = last - 1  # fewer keys than new rows
        nan[c.N - last:] = True
    elif what == "page":
        c.table[-1, 3] = -1
        nan[c.N - last:] = True
    else:
        c.q.view(c.N, H, D)[c.N - 1, H - 1, D // 2] = math.nan
        nan[c.N - 1, H - 1] = True
    out, lse = c.call(zt, workspace=ws)
    ref = [torch.cat(x) for x in zip(*(c.reference(b) for b in range(len(rows))))]
    out, want = out.view(c.N, H, D), ref[0].view(c.N, H, D)
    assert out[nan].isnan().all() and lse[nan].isnan().all()
    if (~nan).any():
        near(out[~nan], want[~nan], "out")
        near(lse[~nan], ref[1][~nan], "lse")
    assert (behind == 255).all() and zt.lib.tc_status() == 0
