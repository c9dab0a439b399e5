"""PagedLayer.set_lens: the host's counts after rows that were written past it."""
import pytest
import torch


def layer(zt, **over):
    return zt.kv_cache.PagedLayer(**{"n_pages": 8, "page_size": 4, "width": 8, "batch": 2, "max_pages": 4, "device": "cpu", **over})


def test_counts_whose_rows_have_pages(zt):
    c = layer(zt)
    c.reserve([7, 2])
    c.set_lens([7, 1])
    assert c._len == [7, 1] and c.len.tolist() == [7, 1]
    c.set_lens(torch.tensor([8, 4]))  # the rest of their pages
    c.set_lens([3, 0])  # and back
    c.set_lens([8, 4])
    held, table = c.free_pages(), c.table.clone()
    for bad in ([9, 4], [8, 5], [17, 0], [-1, 0], [1], [1, 1, 1], [[1, 1]]):
        with pytest.raises(zt.ops.DimensionMismatch):
            c.set_lens(bad)
        assert c._len == [8, 4] and c.len.tolist() == [8, 4]
    assert c.free_pages() == held and torch.equal(c.table, table)
    c.reserve([1, 1])  # the next rows' pages follow from the counts
    assert c.free_pages() == held - 2 and (c.table[:, 2] >= 0).tolist() == [True, False] and (c.table[:, 1] >= 0).all()
    with pytest.raises(zt.kv_cache.Full):
        c.reserve([9, 0])


def test_pages_behind_a_window_may_be_gone(zt):
    c = layer(zt)
    c.reserve([16, 0])
    c.set_lens([12, 0])
    assert c.trim(window=3) == 2  # slots 10 and 11 are seen and 12: pages 0 and 1 go
    c.set_lens([15, 0])
    assert c._len == [15, 0]
    with pytest.raises(zt.ops.DimensionMismatch):  # slots 4 and 5 went with their page, and 6 would share a new one with them
        c.set_lens([6, 0])
    c.set_lens([9, 0])
    assert c._len == [9, 0]


@pytest.mark.gpu
def test_appends_behind_a_graph_s_replays(zt):
    """Steps in a graph, then a chunk through the layer: its rows find the pages behind those that the replays wrote."""
    from test_gpu_paged import Case, near, rand
    H, G, D, page, B = 4, 2, 64, 8, 2
    c = zt.kv_cache.PagedLayer(20, page, G * D, B, 8)
    c.reserve([14, 14])
    k, v, q = (torch.zeros(B, w * D, device="cuda") for w in (G, G, H))
    zt.paged_append(c.k, c.v, c.table, c.len, k, v)  # (a first call outside)
    c.len.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        zt.paged_append(c.k, c.v, c.table, c.len, k, v)
    held = [[], []]
    for i in range(13):
        for x, y, h in zip((k, v), (rand(B, G * D, seed=2 * i), rand(B, G * D, seed=2 * i + 1)), held):
            x.copy_(y), h.append(y)
        graph.replay()
    c.set_lens([13, 13])
    rows = [9, 5]
    kn, vn, qn = (rand(sum(rows), w * D, seed=90 + i) for i, w in enumerate((G, G, H)))
    cu = c.append(kn, vn, rows)
    out, lse = zt.kv_cache.attn_rows(qn, c, H, G, D, cu_rows=cu, want_lse=True)
    assert c.len.tolist() == [22, 18] == c._len and int(c.skipped) == 0
    at = 0
    for b, r in enumerate(rows):
        one = Case.__new__(Case)
        one.rows, one.past, one.H, one.G, one.D, one.window, one.sinks = [r], [13], H, G, D, 0, 0
        one.q, one.cu = qn[at:at + r], torch.tensor([0, r])
        one.keys = [[torch.cat([torch.stack([x[b] for x in h]), new[at:at + r]]) for h, new in zip(held, (kn, vn))]]
        ref, ref_lse = one.reference(0)
        near(out[at:at + r], ref, b)
        near(lse[at:at + r], ref_lse, b)
        at += r
