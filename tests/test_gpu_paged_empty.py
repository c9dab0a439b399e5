"""Paged calls without new rows: what a scheduler issues when no sequence has any."""
import pytest
import torch
from test_gpu_paged import Case

pytestmark = pytest.mark.gpu


def test_a_call_without_rows_counts_no_sequence(zt):
    """Neither what lay in a fresh workspace nor what the call before found."""
    H, G, D, page = 4, 2, 64, 16
    c = Case([5, 6], [20, 30], H, G, D, page, seed=4)
    ws = zt.PagedWorkspace(2, c.N, c.table.shape[1] * page, H, G, D)
    q, cu = c.q[:0], torch.zeros(3, dtype=torch.int32, device="cuda")
    ws.buf.fill_(255)
    n, k = c.n_keys.clone(), c.k.clone()

    def empty():
        zt.paged_append(c.k, c.v, c.table, c.n_keys, c.k.view(-1, G * D)[:0], c.v.view(-1, G * D)[:0], cu_rows=cu)
        return zt.attention_paged(q, c.k, c.v, c.table, c.n_keys, H, G, D, cu_rows=cu, workspace=ws, want_lse=True)

    out, lse = empty()
    assert out.shape == (0, H * D) and lse.shape == (0, H) and ws.bad_sequences() == 0
    assert torch.equal(n, c.n_keys) and torch.equal(k.nan_to_num(7.0), c.k.nan_to_num(7.0))
    c.n_keys[1] = 5  # fewer keys than new rows
    c.call(zt, workspace=ws)
    assert ws.bad_sequences() == 1
    c.n_keys.copy_(n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        empty()
    assert ws.bad_sequences() == 1
    graph.replay()
    assert ws.bad_sequences() == 0
    c.check(*c.call(zt, workspace=ws))
    assert ws.bad_sequences() == 0
