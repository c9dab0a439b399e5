"""Device-resident KV cache with the reference's kv_cache semantics (src/kv_cache.zig).

The reference keeps the cache on the host and re-uploads the whole filled prefix
on every decode step (src/decode.zig:435-437); here the cache lives in HBM, one
[batch, n_ctx, n_kv_heads*head_dim] pair per layer, rows are appended by a kernel
and the decode kernel reads them in place.

A decode loop must not wait for the GPU between steps, so the refusals the reference
makes from a layer's `len` (Error.Full, src/kv_cache.zig:88-95,196) are made here from a
count kept on the host: every append advances every sequence of a layer by one row, so
the host knows an upper bound of the fill counts without reading them back.  Only when
that bound says a sequence MAY be full (lens that were set ragged by hand) are the device
counts read to decide exactly.
"""
from __future__ import annotations

from . import lib as _lib
from .device import ConfigRefused
from .ops import (DecodeWorkspace, DimensionMismatch, PagedWorkspace, _need_cuda_f32, attention_paged, decode_attention,
                  paged_append)


class Full(Exception):
    """kv_cache Error.Full (src/kv_cache.zig:88-95)."""


class Layer:
    """kv_cache.Layer for `batch` sequences: k, v [batch, n_ctx, width] and per-sequence len."""

    def __init__(self, n_ctx: int, width: int, batch: int = 1, device="cuda"):
        import torch
        if n_ctx == 0 or width == 0:
            raise DimensionMismatch("kv_cache.Layer.init")  # src/kv_cache.zig:66
        self.n_ctx, self.width, self.batch = n_ctx, width, batch
        self.k = torch.zeros((batch, n_ctx, width), dtype=torch.float32, device=device)
        self.v = torch.zeros_like(self.k)
        self.len = torch.zeros((batch,), dtype=torch.int32, device=device)
        self._full = torch.zeros((1,), dtype=torch.int32, device=device)
        self._len_bound = 0  # no sequence of the layer holds more rows than this

    def set_lens(self, lens) -> None:
        """Start from given per-sequence fill counts (a ragged batch whose rows were written directly)."""
        import torch
        lens = torch.as_tensor(lens, dtype=torch.int32)
        low, high = map(int, torch.aminmax(lens)) if lens.shape == (self.batch,) else (-1, 0)
        if low < 0 or high > self.n_ctx:
            raise DimensionMismatch("kv_cache.Layer.set_lens")
        self._len_bound = high
        # from ordinary host memory that is ours, the copy has been taken off the host when the call returns: nothing waits
        # for the GPU (given the caller's tensor, pinned perhaps, it would have to)
        self.len.copy_(lens.clone() if lens.device.type == "cpu" else lens, non_blocking=True)

    def check_append(self, k_rows, v_rows) -> None:
        """Every refusal of append, made without writing anything: widths, placement, and Full."""
        if tuple(k_rows.shape) != (self.batch, self.width) or tuple(v_rows.shape) != (self.batch, self.width):
            raise DimensionMismatch("kv_cache.Layer.append")
        _need_cuda_f32(k_rows, v_rows)
        if k_rows.device != self.k.device or v_rows.device != self.k.device:
            raise DimensionMismatch("the new rows must live on the cache's device")
        if self._len_bound >= self.n_ctx:
            # possibly full: the device counts decide (this read waits for the GPU; it happens only at the
            # very end of a cache's life, or on caches whose lens were set ragged)
            if int(self.len.max().item()) >= self.n_ctx:
                raise Full("kv_cache.Layer.append")

    def append(self, k_rows, v_rows) -> None:
        """One new row per sequence ([batch, width]); refuses, writing nothing, when any
        sequence is full or a width is wrong (src/kv_cache.zig:88-95)."""
        if self._len_bound < self.n_ctx and _lib.native().kv_append(self.k, self.v, self.len, k_rows, v_rows, self._full):
            self._len_bound += 1
            return
        self.check_append(k_rows, v_rows)
        self._append_unchecked(k_rows, v_rows)

    def _append_unchecked(self, k_rows, v_rows) -> None:
        import torch
        with torch.cuda.device(self.k.device):
            rc = _lib.load().zt_kv_append(
                self.k.data_ptr(), self.v.data_ptr(), self.len.data_ptr(), k_rows.data_ptr(), v_rows.data_ptr(),
                self._full.data_ptr(), self.batch, self.n_ctx, 1, self.width,
                torch.cuda.current_stream(self.k.device).cuda_stream)
        if rc != 0:
            raise ConfigRefused(_lib.last_error())
        self._len_bound = min(self._len_bound + 1, self.n_ctx)

    def skipped_full(self) -> int:
        """Sequences the append kernel has left untouched because they were full, over the layer's life (reads
        the device: waits for the GPU).  Zero unless a caller bypassed check_append."""
        return int(self._full.item())

    def visible(self):
        """Per-sequence filled row counts (src/kv_cache.zig:133-135)."""
        return self.len

    def bytes(self) -> int:
        return 2 * self.batch * self.n_ctx * self.width * 4


class Cache:
    """kv_cache.Cache (src/kv_cache.zig:140-225): one Layer per transformer layer, advanced together."""

    def __init__(self, n_layers: int, n_ctx: int, width: int, batch: int = 1, device="cuda"):
        if n_layers == 0:
            raise DimensionMismatch("kv_cache.Cache.init")  # src/kv_cache.zig:154
        self.layers = [Layer(n_ctx, width, batch, device) for _ in range(n_layers)]
        self.len = 0

    def append_all(self, ks, vs) -> None:
        """One position for every layer, all or nothing (src/kv_cache.zig:180-200): EVERY layer is checked
        (count of tensors, widths, room) before ANY of them is written."""
        if len(ks) != len(self.layers) or len(vs) != len(self.layers):
            raise DimensionMismatch("kv_cache.Cache.appendAll")
        for layer, k_rows, v_rows in zip(self.layers, ks, vs):
            layer.check_append(k_rows, v_rows)
        for layer, k_rows, v_rows in zip(self.layers, ks, vs):
            layer._append_unchecked(k_rows, v_rows)
        self.len += 1

    def full(self) -> bool:
        """Whether another position would not fit (src/kv_cache.zig:211-214)."""
        if not self.layers:
            return True
        return self.len >= self.layers[0].n_ctx

    def bytes(self) -> int:
        """src/kv_cache.zig:220-224."""
        return sum(layer.bytes() for layer in self.layers)


def attn_step(q, layer: Layer, n_heads, n_kv_heads, head_dim, *, workspace: DecodeWorkspace | None = None,
              want_lse=False):
    """decode.cudaAttnStep (src/decode.zig:405-473) without the per-step upload: q [batch, H*D]."""
    if layer.width != n_kv_heads * head_dim:
        raise DimensionMismatch("cache width disagrees with the head configuration")
    return decode_attention(q, layer.k, layer.v, layer.len, n_heads, n_kv_heads, head_dim,
                            workspace=workspace, want_lse=want_lse)


class PagedLayer:
    """A layer's cache for `batch` sequences whose rows lie in pages of a common pool: k, v [n_pages, page_size, width], a table
    [batch, max_pages] of every sequence's pages (-1: none) and per-sequence len.  Which pages are whose is decided on the host, from
    counts kept there; no step reads the device.  So what changes them is refused inside a stream capture, whose replays would not: a graph
    calls paged_append and attn_rows, over pages that reserve() has found beforehand, and set_lens() says afterwards how far it went.  (kv_cache.Layer, src/kv_cache.zig:60-135, keeps n_ctx rows for each.)"""

    def __init__(self, n_pages: int, page_size: int, width: int, batch: int, max_pages: int, device="cuda"):
        import torch
        if min(n_pages, page_size, width, batch, max_pages) < 1 or width % 4 != 0:
            raise DimensionMismatch("kv_cache.PagedLayer")
        self.n_pages, self.page_size, self.width, self.batch, self.max_pages = n_pages, page_size, width, batch, max_pages
        self.k = torch.zeros((n_pages, page_size, width), dtype=torch.float32, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.len = torch.zeros((batch,), dtype=torch.int32, device=device)
        self.skipped = torch.zeros((1,), dtype=torch.int32, device=device)
        self._table = torch.full((batch, max_pages), -1, dtype=torch.int32)
        self._len = [0] * batch
        self._free = list(range(n_pages - 1, -1, -1))

    def free_pages(self) -> int:
        return len(self._free)

    def _decides(self, what):
        import torch
        if self.k.is_cuda and torch.cuda.is_current_stream_capturing():
            raise ConfigRefused(f"kv_cache.PagedLayer.{what} decides on the host: a captured one would not when it is replayed")

    def _send_table(self):
        # (a copy that is ours alone: the host's table may change before the device has read it)
        self.table.copy_(self._table.clone(), non_blocking=True)

    def append(self, k_rows, v_rows, counts=None):
        """counts[b] new rows of each sequence, behind one another in k_rows, v_rows [N, width] (None: one each).  Refuses with
        Full, writing nothing, when a sequence has no place left in the table or the pool no page.  Returns the rows' bounds
        cu_rows on the device (None for one row each), which attn_rows takes."""
        import torch
        self._decides("append")
        given = [1] * self.batch if counts is None else [int(n) for n in counts]
        if len(given) != self.batch or min(given) < 0:
            raise DimensionMismatch("kv_cache.PagedLayer.append takes a count for every sequence")
        shape = (sum(given), self.width)
        if tuple(k_rows.shape) != shape or tuple(v_rows.shape) != shape:
            raise DimensionMismatch("kv_cache.PagedLayer.append")
        _need_cuda_f32(k_rows, v_rows)
        if k_rows.device != self.k.device or v_rows.device != self.k.device:
            raise DimensionMismatch("the new rows must live on the cache's device")
        self.reserve(given)
        cu = None
        if counts is not None:
            cu = torch.zeros(self.batch + 1, dtype=torch.int32)
            cu[1:] = torch.tensor(given, dtype=torch.int32).cumsum(0)
            cu = cu.to(self.k.device, non_blocking=True)
        paged_append(self.k, self.v, self.table, self.len, k_rows, v_rows, cu_rows=cu, skipped=self.skipped)
        self._len = [n + m for n, m in zip(self._len, given)]
        return cu

    def set_lens(self, lens) -> None:
        """Start from given per-sequence fill counts: rows were written directly, or by the replays of a captured paged_append, of which the host's
        counts know nothing.  Refuses a count whose rows lie beyond the table or, behind those that were known, on no page."""
        import torch
        self._decides("set_lens")
        lens = torch.as_tensor(lens, dtype=torch.int32)
        given = lens.tolist() if lens.shape == (self.batch,) else [-1]
        if min(given) < 0 or max(given) > self.max_pages * self.page_size:
            raise DimensionMismatch("kv_cache.PagedLayer.set_lens")
        for b, n in enumerate(given):
            new = self._table[b, self._len[b] // self.page_size:-(-n // self.page_size)]
            # (going back, the page that the next row shares with older ones has to be there still)
            shared = n % self.page_size > 0 and int(self._table[b, n // self.page_size]) < 0
            if shared or n > self._len[b] and bool((new < 0).any()):
                raise DimensionMismatch("kv_cache.PagedLayer.set_lens: rows on no page")
        self._len = given
        self.len.copy_(torch.tensor(given, dtype=torch.int32), non_blocking=True)  # (host memory of its own: see Layer.set_lens)

    def reserve(self, counts) -> None:
        """Pages for counts[b] more rows of each sequence, for all of them or (Full) for none."""
        self._decides("reserve")
        counts, wanted = list(counts), []
        if len(counts) != self.batch:
            raise DimensionMismatch("kv_cache.PagedLayer.reserve takes a count for every sequence")
        for b, n in enumerate(counts):
            if n < 0:
                raise DimensionMismatch("kv_cache.PagedLayer.reserve")
            if self._len[b] + n > self.max_pages * self.page_size:
                raise Full("kv_cache.PagedLayer: the sequence's table")
            wanted += [(b, s) for s in range(self._len[b] // self.page_size, -(-(self._len[b] + n) // self.page_size))
                       if self._table[b, s] < 0]
        if len(wanted) > len(self._free):
            raise Full("kv_cache.PagedLayer: the pool")
        for b, s in wanted:
            self._table[b, s] = self._free.pop()
        if wanted:
            self._send_table()

    def release(self, b: int) -> None:
        """The sequence ends: its pages go back to the pool and its place is empty again."""
        self._decides("release")
        self._give_back(b, range(self.max_pages))
        self._len[b] = 0
        self.len[b].zero_()

    def trim(self, window: int, sinks: int = 0) -> int:
        """Gives back the pages that no coming query of `window` and `sinks` sees; returns how many."""
        if window < 1 or sinks < 0:
            raise DimensionMismatch("kv_cache.PagedLayer.trim")
        self._decides("trim")
        before, ps = len(self._free), self.page_size
        for b, n in enumerate(self._len):
            # the next query stands at n and sees slots from n - window + 1 on
            self._give_back(b, range(-(-sinks // ps), max(0, n - window + 1) // ps))
        return len(self._free) - before

    def _give_back(self, b, slots) -> None:
        held = [s for s in slots if self._table[b, s] >= 0]
        self._free += [int(self._table[b, s]) for s in held]
        self._table[b, held] = -1
        if held:
            self._send_table()

    def bytes(self) -> int:
        return 2 * self.n_pages * self.page_size * self.width * 4


def attn_rows(q, layer: PagedLayer, n_heads, n_kv_heads, head_dim, *, cu_rows=None, window=0, sinks=0,
              workspace: PagedWorkspace | None = None, want_lse=False):
    """attn_step over pages, for the rows that layer.append took last (and whose bounds it returned): q [N, H*D]."""
    if layer.width != n_kv_heads * head_dim:
        raise DimensionMismatch("cache width disagrees with the head configuration")
    return attention_paged(q, layer.k, layer.v, layer.table, layer.len, n_heads, n_kv_heads, head_dim, cu_rows=cu_rows,
                           window=window, sinks=sinks, workspace=workspace, want_lse=want_lse)
