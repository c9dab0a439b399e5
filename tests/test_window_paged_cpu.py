"""Attention with a window and sinks, and over a paged cache, as far as no GPU is needed: refusals of the C entry points and of
the Python calls, and which pages the paged cache's host side hands out."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(256)  # never dereferenced: every case is refused before any launch


@pytest.fixture
def L(zt):
    lib = zt.lib.load()
    lib.zt_attn_set_verbose(0)
    yield lib
    lib.zt_attn_set_verbose(1)


@pytest.mark.parametrize("over,fragment", [
    (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(B=0), "batch 0"), (dict(B=65536), "batch 65536"),
    (dict(T=0), "T 0"), (dict(D=33), "head_dim 33"), (dict(H=5), "not a group"),
])
def test_window_calls_refuse(zt, L, over, fragment):
    a = {"B": 1, "T": 8, "H": 4, "G": 2, "D": 32, "window": 4, "sinks": 1, **over}
    shape = [a[x] for x in ("B", "T", "H", "G", "D", "window", "sinks")]
    assert L.zt_attn_forward_window_batched(*[ONE] * 5, *shape, None) == 1 and fragment in zt.lib.last_error()
    assert L.zt_attn_backward_window_batched(*[ONE] * 11, 1 << 30, *shape, None) == 1 and fragment in zt.lib.last_error()


def test_window_calls_refuse_null_pointers_and_short_workspaces(zt, L):
    assert L.zt_attn_forward_window_batched(ONE, None, ONE, ONE, None, 1, 8, 4, 2, 32, 4, 0, None) == 1 and "null" in zt.lib.last_error()
    assert L.zt_attn_backward_window_batched(*[ONE] * 10, None, 0, 1, 256, 4, 2, 64, 4, 0, None) == 1
    assert "workspace" in zt.lib.last_error()


def paged(L, **over):
    a = {"q": ONE, "k": ONE, "v": ONE, "table": ONE, "n_keys": ONE, "cu": ONE, "out": ONE, "lse": None, "ws": ONE, "bytes": 1 << 40, "B": 2,
         "rows": 3, "n_pages": 4, "page": 16, "max_pages": 2, "H": 4, "G": 2, "D": 32, "window": 0, "sinks": 0, **over}
    return L.zt_attn_paged(*a.values(), None)


@pytest.mark.parametrize("over,fragment", [
    (dict(B=0), "batch 0"), (dict(n_pages=0), "not a cache"), (dict(page=0), "not a cache"), (dict(max_pages=0), "not a cache"),
    (dict(max_pages=1 << 20, page=1 << 12), "not a cache"), (dict(D=34), "multiples of four"), (dict(D=30), "head_dim 30"),
    (dict(H=5), "not a group"), (dict(rows=-1), "rows"), (dict(cu=None), "cu_rows"), (dict(q=None), "null"), (dict(table=None), "null"),
    (dict(window=-2), "window"), (dict(sinks=-2), "sinks"), (dict(ws=None), "workspace"), (dict(bytes=16), "workspace"),
    (dict(ws=ctypes.c_void_p(264)), "256-byte"), (dict(q=ctypes.c_void_p(260)), "16-byte"), (dict(v=ctypes.c_void_p(264)), "16-byte"),
    (dict(out=ctypes.c_void_p(4)), "16-byte"),
])
def test_paged_attention_refuses(zt, L, over, fragment):
    assert paged(L, **over) == 1 and fragment in zt.lib.last_error()


@pytest.mark.parametrize("over,fragment", [
    (dict(B=0), "batch 0"), (dict(n_pages=0), "not a cache"), (dict(width=30), "multiple of four"), (dict(rows=-1), "rows"),
    (dict(cu=None), "cu_rows"), (dict(k_new=None), "null"), (dict(n_keys=None), "null"), (dict(v_new=ctypes.c_void_p(24)), "16-byte"),
])
def test_paged_append_refuses(zt, L, over, fragment):
    a = {"k": ONE, "v": ONE, "table": ONE, "n_keys": ONE, "k_new": ONE, "v_new": ONE, "cu": ONE, "skipped": None, "B": 2, "rows": 3,
         "n_pages": 4, "page": 16, "max_pages": 2, "width": 64, **over}
    assert L.zt_kv_append_paged(*a.values(), None) == 1 and fragment in zt.lib.last_error()


def test_paged_workspace_size(zt, L):
    size = L.zt_attn_paged_workspace_bytes
    assert size(0, 1, 16, 4, 2, 32) == size(1, -1, 16, 4, 2, 32) == size(1, 1, 0, 4, 2, 32) == size(1, 1, 16, 4, 3, 32) == size(1, 1, 16, 4, 2, 34) == 0
    # a workspace serves every smaller call: it does not shrink as any of its numbers grows
    for H, G, D in ((32, 8, 128), (4, 2, 32), (16, 16, 64), (8, 2, 256), (12, 4, 96)):
        last = 0
        for n in (1, 2, 3, 16, 64, 128, 129, 300, 1000, 4000):
            now = size(n, n, 20000, H, G, D)
            assert now >= last > -1
            last = now
        for keys in (1, 100, 1000, 30000):
            worst = max(size(b, r, k, H, G, D) for b in (1, 2, 5) for r in (1, 2, 5, 77, 200) for k in (1, 50, keys))
            assert size(5, 200, keys if keys > 50 else 50, H, G, D) >= worst


@pytest.mark.parametrize("H,G,D", [(32, 8, 128), (4, 2, 32), (16, 16, 64), (8, 2, 256), (12, 4, 96), (64, 1, 64), (300, 1, 32)])
def test_paged_workspace_holds_a_step_over_any_part_of_the_keys(zt, L, H, G, D):
    """A step over a window is planned for the keys that it sees: the plan of every smaller step fits."""
    for B in (1, 2, 7, 30, 64, 300):
        for keys in (1, 64, 129, 1000, 2047, 6145, 20000, 131072):
            room = L.zt_attn_paged_workspace_bytes(B, B, keys, H, G, D)
            for n in {keys, *(k for k in (1, 100, 128, 500, 769, 1025, 3000, 8000, 16385, 100000) if k < keys)}:
                for b in {B, max(1, B // 2), 1}:
                    assert L.zt_attn_decode_workspace_bytes(b, n, H, G, D) <= room, (b, n, keys)


def test_python_calls_refuse_what_is_not_on_a_gpu(zt):
    x = torch.zeros(1, 4, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        zt.attention_forward_window(x, x, x, 2, 2, 32, 2)
    with pytest.raises(zt.ops.InvalidHeadConfig):
        zt.attention_forward_window(x, x, x, 3, 2, 32, 2)
    pages = torch.zeros(2, 4, 64)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        zt.paged_append(pages, pages, table, n, x[0, :1], x[0, :1])
    with pytest.raises(RuntimeError, match="no CPU path"):
        zt.attention_paged(x[0, :1], pages, pages, table, n, 2, 2, 32)


def layer(zt, **over):
    return zt.kv_cache.PagedLayer(**{"n_pages": 6, "page_size": 4, "width": 8, "batch": 2, "max_pages": 4, "device": "cpu", **over})


def test_pages_are_handed_out_once_and_all_or_nothing(zt):
    c = layer(zt)
    c.reserve([5, 4])
    assert c.free_pages() == 3 and (c.table >= 0).sum(1).tolist() == [2, 1]
    held = c.table[c.table >= 0].tolist()
    assert len(set(held)) == 3 and all(0 <= x < 6 for x in held)
    c._len = [5, 4]
    before = c.table.clone()
    for counts in ([12, 0], [11, 9]):  # beyond the table; beyond the pool
        with pytest.raises(zt.kv_cache.Full):
            c.reserve(counts)
        assert torch.equal(c.table, before) and c.free_pages() == 3
    c.reserve([3, 0])  # the second page has room
    assert c.free_pages() == 3
    for counts in ([1], [1, 0, 1], [1, -1]):
        with pytest.raises(zt.ops.DimensionMismatch):
            c.reserve(counts)
        assert c.free_pages() == 3
    c.reserve([11, 0])
    assert c.free_pages() == 1
    c._len = [16, 4]
    c.release(0)
    assert c.free_pages() == 5 and c.table[0].tolist() == [-1] * 4 and c._len == [0, 4]


def test_trim_keeps_what_a_coming_query_sees(zt):
    c = layer(zt, n_pages=20, batch=3, max_pages=10)
    c.reserve([40, 13, 3])
    c._len = [40, 13, 3]
    table = c.table.clone()
    assert c.trim(window=9, sinks=5) == 6  # slots 32 .. 40 are seen and 0 .. 4: pages 2 .. 7 of the first go
    assert [s for s in range(10) if c.table[0, s] >= 0] == [0, 1, 8, 9]
    assert torch.equal(c.table[1:], table[1:])
    assert c.trim(window=2) == 3 + 3  # 39 and 40 are seen of the first, 12 and 13 of the second
    assert [s for s in range(10) if c.table[0, s] >= 0] == [9]
    assert [s for s in range(10) if c.table[1, s] >= 0] == [3]
    with pytest.raises(zt.ops.DimensionMismatch):
        c.trim(0)


@pytest.mark.parametrize("over", [dict(n_pages=0), dict(page_size=0), dict(width=0), dict(width=6), dict(batch=0), dict(max_pages=0)])
def test_degenerate_paged_layers_are_refused(zt, over):
    with pytest.raises(zt.ops.DimensionMismatch):
        layer(zt, **over)
