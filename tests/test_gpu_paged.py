"""A paged cache: the append of new rows and their attention, against the formulas in 64 bits (tolerance and its reasons: test_gpu_window.py,
sums of up to 7000 keys here, whose weights are smaller for it)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NAN = float("nan")


def rand(*shape, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda")


class Case:
    """Sequences of rows[b] new rows behind past[b] old ones, on pages in no order; what no query may read is NaN."""

    def __init__(self, rows, past, H, G, D, page, window=0, sinks=0, seed=0, extra=0):
        self.rows, self.past, self.H, self.G, self.D, self.page, self.window, self.sinks = rows, past, H, G, D, page, window, sinks
        B, keys = len(rows), [r + n for r, n in zip(rows, past)]
        used = [-(-n // page) for n in keys]
        host = torch.Generator()
        host.manual_seed(seed)
        order = torch.randperm(sum(used) + 2, generator=host).int()
        self.table = torch.full((B, max(1, *used, 1)), -1, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = order[at:at + u]
            at += u
        self.table = self.table.cuda()
        self.n_keys = torch.tensor(keys, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor([0, *rows], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
        self.N = sum(rows) + extra
        self.q = rand(self.N, H * D, seed=seed + 1)
        self.k, self.v = (torch.full((len(order), page, G * D), NAN, device="cuda") for _ in range(2))
        self.keys = [[rand(n, G * D, seed=seed + 10 + 2 * b + i) for i in range(2)] for b, n in enumerate(keys)]
        for b, n in enumerate(keys):
            j = torch.arange(n, device="cuda")
            if window:  # (the pages of the others might be anyone's)
                j = j[(j > past[b] - window) | (j < sinks)]
            ids = self.table[b].long()[j // page]
            self.k[ids, j % page], self.v[ids, j % page] = self.keys[b][0][j], self.keys[b][1][j]

    def reference(self, b):
        H, G, D, r, n = self.H, self.G, self.D, self.rows[b], self.past[b]
        q = self.q[int(self.cu[b]):int(self.cu[b]) + r].double().view(r, G, H // G, D)
        k, v = (x.double().view(-1, G, D) for x in self.keys[b])
        pos, j = torch.arange(n, n + r, device="cuda")[:, None], torch.arange(n + r, device="cuda")[None, :]
        hidden = j > pos
        if self.window:
            hidden = hidden | ((j <= pos - self.window) & (j >= self.sinks))
        s = (torch.einsum("tgrd,sgd->grts", q, k) / math.sqrt(D)).masked_fill(hidden, -math.inf)
        lse = torch.logsumexp(s, -1)
        out = torch.einsum("grts,sgd->tgrd", torch.exp(s - lse[..., None]), v)
        return out.reshape(r, H * D), lse.permute(2, 0, 1).reshape(r, H)

    def call(self, zt, **kw):
        return zt.attention_paged(self.q, self.k, self.v, self.table, self.n_keys, self.H, self.G, self.D, cu_rows=self.cu,
                                  window=self.window, sinks=self.sinks, want_lse=True, **kw)

    def check(self, out, lse, skip=()):
        for b, r in enumerate(self.rows):
            if r == 0 or b in skip:
                continue
            at = slice(int(self.cu[b]), int(self.cu[b]) + r)
            for got, ref in zip((out[at], lse[at]), self.reference(b)):
                near(got, ref, b)


def near(got, ref, what):
    err = (got.double() - ref).abs() - (1e-5 + 1e-4 * ref.abs())
    assert torch.isfinite(got).all() and err.max() <= 0, (what, float((got.double() - ref).abs().max()), float(err.max()))


CHUNKS = [
    # rows, past, H, G, D, page, window, sinks: the smallest
    ([1], [0], 2, 1, 32, 1, 0, 0), ([2], [0], 4, 2, 64, 16, 0, 0), ([3, 1, 2], [0, 5, 1], 4, 2, 64, 4, 0, 0),
    # sequences without new rows between others, pages that end inside a tile, one-row pages
    ([0, 5, 0, 0, 7, 0], [3, 60, 0, 9, 64, 1], 8, 2, 64, 7, 0, 0), ([40], [100], 4, 4, 32, 1, 0, 0), ([33, 65], [63, 127], 4, 1, 64, 50, 0, 0),
    # many rows, few keys; few rows, many keys
    ([300], [0], 4, 2, 64, 16, 0, 0), ([5], [3000], 8, 2, 64, 16, 0, 0), ([2, 17], [6000, 700], 32, 8, 128, 64, 0, 0), ([77], [923], 32, 8, 128, 16, 0, 0),
    ([600, 1, 130], [200, 2000, 0], 4, 2, 128, 300, 0, 0),
    # windows, sinks
    ([1, 9], [50, 400], 4, 2, 64, 16, 1, 0), ([40, 200], [500, 90], 8, 2, 64, 16, 64, 4), ([40, 200], [500, 90], 8, 2, 64, 10, 33, 70),
    ([129], [1000], 4, 2, 128, 64, 300, 1), ([20, 3], [10, 0], 4, 2, 32, 8, 100, 4), ([64], [5000], 16, 16, 64, 32, 2048, 16),
    # widths and groups
    ([50, 20], [100, 300], 6, 2, 96, 16, 0, 0), ([45], [211], 16, 4, 80, 16, 40, 3), ([45], [211], 5, 1, 100, 16, 0, 0), ([30, 30], [64, 0], 12, 4, 36, 9, 0, 0),
    ([70], [200], 4, 2, 256, 16, 0, 0), ([33, 1], [90, 700], 8, 2, 192, 32, 64, 4), ([40], [600], 8, 1, 160, 16, 0, 0), ([20], [99], 3, 3, 252, 5, 50, 2),
    ([100], [50], 64, 1, 64, 16, 0, 0), ([9], [500], 1, 1, 128, 16, 0, 0), ([3], [20], 300, 1, 32, 16, 0, 0),
]


@pytest.mark.parametrize("rows,past,H,G,D,page,window,sinks", CHUNKS)
def test_chunks(zt, rows, past, H, G, D, page, window, sinks):
    c = Case(rows, past, H, G, D, page, window, sinks, seed=len(rows) + D + page)
    ws = zt.PagedWorkspace(len(rows), c.N, c.table.shape[1] * page, H, G, D)
    ws.buf.fill_(255)
    out, lse = c.call(zt, workspace=ws)
    again, lse2 = c.call(zt)
    c.check(out, lse)
    assert ws.bad_sequences() == 0 and torch.equal(out, again) and torch.equal(lse, lse2)
    assert zt.lib.tc_status() == 0


STEPS = [
    # past, H, G, D, page, window, sinks
    ([0], 2, 1, 32, 1, 0, 0), ([0, 1, 2, 15, 16, 17], 4, 2, 64, 16, 0, 0), ([999], 32, 8, 128, 16, 0, 0), ([7000, 3, 500], 32, 8, 128, 64, 0, 0),
    ([6500], 8, 2, 64, 50, 0, 0), ([100] * 40, 8, 8, 64, 8, 0, 0), ([37 * i % 900 for i in range(70)], 16, 4, 128, 16, 0, 0),
    ([500, 3, 64, 65, 4000], 8, 2, 128, 16, 64, 4), ([500, 0, 9], 4, 4, 96, 7, 1, 0), ([800, 100], 4, 1, 80, 16, 33, 50), ([3000] * 20, 4, 2, 64, 64, 700, 16),
    ([300, 2000], 8, 1, 256, 16, 0, 0), ([300, 20], 6, 2, 192, 32, 100, 1), ([77, 5], 4, 2, 36, 3, 0, 0), ([1000] * 12, 12, 4, 160, 16, 512, 4),
]


@pytest.mark.parametrize("past,H,G,D,page,window,sinks", STEPS)
def test_steps(zt, past, H, G, D, page, window, sinks):
    """One new row a sequence: with and without its bounds spelt out."""
    c = Case([1] * len(past), past, H, G, D, page, window, sinks, seed=len(past) + D)
    out, lse = zt.attention_paged(c.q, c.k, c.v, c.table, c.n_keys, H, G, D, window=window, sinks=sinks, want_lse=True)
    c.check(out, lse)
    c.check(*c.call(zt))
    given = torch.full_like(c.q, 9.0)
    assert zt.attention_paged(c.q, c.k, c.v, c.table, c.n_keys, H, G, D, window=window, sinks=sinks, out=given) is given and torch.equal(given, out)


@pytest.mark.parametrize("D,rows", [(64, [40, 3, 70]), (128, [1, 1, 1]), (256, [5, 2, 30])])
def test_rows_behind_the_last_sequence_are_left_as_they_were(zt, D, rows):
    H, G = 8, 2
    c = Case(rows, [100, 7, 900], H, G, D, 16, seed=3, extra=150)
    out = torch.full_like(c.q, 9.0)
    got, lse = c.call(zt, out=out)
    assert got is out and (out[sum(rows):] == 9.0).all()
    c.check(out, lse)


@pytest.mark.parametrize("D", [64, 256])
def test_contradictory_counts_are_nan_rows_and_counted(zt, D):
    H, G, rows = 4, 2, [5, 6, 7, 8]
    c = Case(rows, [20, 30, 40, 50], H, G, D, 16, seed=4)
    ws = zt.PagedWorkspace(4, c.N, c.table.shape[1] * 16, H, G, D)
    c.n_keys[1], c.n_keys[3] = 5, c.table.shape[1] * 16 + 1  # fewer keys than new rows; more than the table holds
    out, lse = c.call(zt, workspace=ws)
    assert ws.bad_sequences() == 2
    for b in (1, 3):
        at = slice(int(c.cu[b]), int(c.cu[b + 1]))
        assert out[at].isnan().all() and lse[at].isnan().all()
    c.check(out, lse, skip=(1, 3))


def test_contradictory_counts_of_steps(zt):
    H, G, D = 4, 2, 64
    c = Case([1] * 5, [10, 20, 30, 40, 50], H, G, D, 16, seed=4)
    ws = zt.PagedWorkspace(5, 5, c.table.shape[1] * 16, H, G, D)
    c.n_keys[0], c.n_keys[2], c.n_keys[4] = 0, -3, 4097
    out, lse = zt.attention_paged(c.q, c.k, c.v, c.table, c.n_keys, H, G, D, workspace=ws, want_lse=True)
    assert ws.bad_sequences() == 3
    assert out[::2].isnan().all() and lse[::2].isnan().all()
    c.check(out, lse, skip=(0, 2, 4))


def test_bounds_that_do_not_ascend_or_leave_the_tensor(zt):
    H, G, D = 4, 2, 64
    c = Case([5, 5, 5], [20, 20, 20], H, G, D, 16, seed=6)
    ws = zt.PagedWorkspace(3, c.N, c.table.shape[1] * 16, H, G, D)
    for bounds, bad in (([0, 5, 10, 99], 1), ([0, 5, 3, 15], 1), ([-4, 5, 10, 15], 1)):
        c.cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        out, lse = c.call(zt, workspace=ws)
        assert ws.bad_sequences() == bad, bounds


@pytest.mark.parametrize("D,rows", [(64, 12), (128, 1), (256, 12), (128, 150)])
@pytest.mark.parametrize("number", [-1, 10**6, -2**31])
def test_rows_that_see_a_page_that_is_none_are_nan(zt, D, rows, number):
    """And no others: the rows before it, those whose window has passed it, other sequences."""
    H, G, page, window = 8, 2, 16, 40
    for r, past, hole in ((rows, 100, 5), (rows, 100, 6)):
        c = Case([r, 3], [past, 30], H, G, D, page, window, 2, seed=9)
        c.table[0, hole] = number
        out, lse = c.call(zt)
        pos = torch.arange(past, past + r, device="cuda")
        slots = torch.arange(hole * page, (hole + 1) * page, device="cuda")
        hit = ((slots[None, :] <= pos[:, None]) & (slots[None, :] > pos[:, None] - window)).any(1)
        assert out[:r][hit].isnan().all() and lse[:r][hit].isnan().all()
        ref, ref_lse = c.reference(0)
        if (~hit).any():
            near(out[:r][~hit], ref[~hit], "out")
            near(lse[:r][~hit], ref_lse[~hit], "lse")
        c.check(out, lse, skip=(0,))


@pytest.mark.parametrize("D,G", [(64, 2), (128, 4), (256, 2), (80, 2)])
@pytest.mark.parametrize("rows", [1, 40, 150])
def test_what_is_not_finite_reaches_the_rows_that_see_it_and_no_others(zt, D, G, rows):
    H, past, window = 2 * G, 300, 64
    for where, value in (("v", NAN), ("v", math.inf), ("v", -math.inf), ("k", NAN)):
        c = Case([rows], [past], H, G, D, 16, window, 3, seed=11)
        j, col = past - 20, D + 5  # an old key that some rows see and later ones do not; a column of KV head 1
        i = 0 if where == "k" else 1
        c.keys[0][i][j, col] = value
        page = c.table[0, j // 16]
        (c.k if where == "k" else c.v)[page, j % 16, col] = value
        out, lse = c.call(zt)
        out, lse = out.view(rows, H, D), lse.view(rows, H)
        ref, ref_lse = (x.view(rows, H, -1).squeeze(-1) for x in c.reference(0))
        hit = torch.arange(past, past + rows, device="cuda") - window < j
        group = torch.arange(H, device="cuda") // (H // G) == 1
        if where == "k":
            assert out[hit][:, group].isnan().all() and lse[hit][:, group].isnan().all()
            clean = ~(hit[:, None] & group[None, :])
            near(out[clean], ref[clean], "out")
            near(lse[clean], ref_lse[clean], "lse")
        else:
            spoilt = hit[:, None, None] & group[None, :, None] & (torch.arange(D, device="cuda") == 5)[None, None, :]
            got = out[spoilt]
            assert (got.isnan().all() if math.isnan(value) else (got == value).all())
            clean = clean64(c, where, i, j, col)
            near(out[~spoilt], clean[0].view(rows, H, D)[~spoilt], "out")
            near(lse, clean[1].view(rows, H), "lse")


def clean64(c, where, i, j, col):
    """The reference with that value's place at zero, which the other columns do not notice."""
    old = c.keys[0][i][j, col].clone()
    c.keys[0][i][j, col] = 0.0
    got = c.reference(0)
    c.keys[0][i][j, col] = old
    return got


@pytest.mark.parametrize("scale", [1e-12, 1e6])
def test_magnitudes(zt, scale):
    """Outputs go with v's size, scores with q's and k's product; tolerance relative to the largest output."""
    c = Case([90], [200], 8, 2, 64, 16, seed=12)
    for x in (c.v, c.keys[0][1]):
        x.mul_(scale)
    for x in (c.k, c.keys[0][0]):
        x.mul_(scale)
    c.q.div_(scale)
    out, lse = c.call(zt)
    ref, ref_lse = c.reference(0)
    near(out / scale, ref / scale, "out")
    near(lse, ref_lse, "lse")


def test_append(zt):
    """New rows of several sequences into their slots, and nothing else; sequences that do not fit are left alone."""
    G, D, page, B = 2, 32, 5, 6
    rows, filled = [3, 0, 7, 1, 12, 4], [0, 4, 9, 4, 14, 6]
    table = torch.full((B, 4), -1, dtype=torch.int32)
    table[:, :] = torch.randperm(24).view(6, 4).int()
    table[3, 0] = -1  # sequence 3's row would lie there: it does not fit
    table[5, 1:] = 99
    cu = torch.tensor([0, *rows], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    N = sum(rows)
    kn, vn = rand(N + 3, G * D, seed=1), rand(N + 3, G * D, seed=2)
    kp, vp = rand(24, page, G * D, seed=3), rand(24, page, G * D, seed=4)
    want_k, want_v, n = kp.clone(), vp.clone(), torch.tensor(filled, dtype=torch.int32, device="cuda")
    fits = [True, True, True, False, False, False]  # 14 + 12 are more than 4 pages of 5
    for b in range(B):
        for i in range(rows[b] if fits[b] else 0):
            s = filled[b] + i
            want_k[table[b, s // page], s % page], want_v[table[b, s // page], s % page] = kn[int(cu[b]) + i], vn[int(cu[b]) + i]
    skipped = torch.zeros(1, dtype=torch.int32, device="cuda")
    zt.paged_append(kp, vp, table.cuda(), n, kn, vn, cu_rows=cu, skipped=skipped)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v) and int(skipped) == 3
    assert n.tolist() == [f + r if ok else f for f, r, ok in zip(filled, rows, fits)]
    # one row each
    filled = [0, 19, 20, 7, -1, 3]
    table[3, 1] = 30
    n.copy_(torch.tensor(filled, dtype=torch.int32))
    zt.paged_append(kp, vp, table.cuda(), n, kn[:B].clone(), vn[:B].clone(), skipped=skipped)
    for b, ok in enumerate([True, True, False, False, False, True]):
        if ok:
            want_k[table[b, filled[b] // page], filled[b] % page], want_v[table[b, filled[b] // page], filled[b] % page] = kn[b], vn[b]
        assert int(n[b]) == filled[b] + ok
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v) and int(skipped) == 6


def test_append_takes_bounds_that_contradict_the_rows(zt):
    kp = torch.zeros(4, 4, 32, device="cuda")
    vp, table, n = torch.zeros_like(kp), torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.zeros(2, dtype=torch.int32, device="cuda")
    kn, skipped = rand(3, 32, seed=1), torch.zeros(1, dtype=torch.int32, device="cuda")
    for bounds, count in (([0, 2, 9], [2, 0]), ([0, -1, 3], [0, 0]), ([0, 2, 1], [2, 0])):
        n.zero_(), kp.zero_(), vp.zero_()
        zt.paged_append(kp, vp, table, n, kn, kn, cu_rows=torch.tensor(bounds, dtype=torch.int32, device="cuda"), skipped=skipped)
        assert n.tolist() == count
        assert torch.equal(kp[0, :count[0]], kn[:count[0]]) and (kp[0, count[0]:] == 0).all() and (kp[1:] == 0).all()


def test_python_refusals(zt):
    c = Case([2, 3], [10, 4], 4, 2, 32, 8, seed=1)
    E = zt.ops
    args = [c.q, c.k, c.v, c.table, c.n_keys, 4, 2, 32]
    for i, bad in ((0, c.q[:, :64]), (0, c.q.half()), (1, c.k[:, :4].contiguous()), (3, c.table.long()), (3, c.table[0]), (4, c.n_keys[:1]), (7, 16), (3, c.table.cpu())):
        with pytest.raises((E.DimensionMismatch, E.InvalidHeadConfig)):
            zt.attention_paged(*[bad if j == i else x for j, x in enumerate(args)], cu_rows=c.cu)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_paged(*args, cu_rows=c.cu[:2])
    with pytest.raises(E.ConfigRefused):
        zt.attention_paged(*args)  # five rows of two sequences
    with pytest.raises(E.ConfigRefused):
        zt.attention_paged(*args, cu_rows=c.cu, window=-1)
    with pytest.raises(E.DimensionMismatch):
        zt.paged_append(c.k, c.v, c.table, c.n_keys, c.q[:, :32].contiguous(), c.q[:, :32].contiguous(), cu_rows=c.cu)
    empty = torch.empty(0, 4 * 32, device="cuda")
    out = zt.attention_paged(empty, c.k, c.v, c.table, c.n_keys, 4, 2, 32, cu_rows=torch.zeros_like(c.cu))
    assert out.shape == (0, 128)


def test_a_paged_layer_over_a_conversation(zt):
    """Prompts, then steps, a window whose pages are given back as they leave it, a sequence that ends and another in its place: at
    every call the attention of all rows so far."""
    H, G, D, page, B, window, sinks = 8, 2, 64, 16, 3, 96, 4
    layer = zt.kv_cache.PagedLayer(40, page, G * D, B, 30)
    layer.k.fill_(NAN), layer.v.fill_(NAN)
    held = [[torch.empty(0, G * D, device="cuda")] * 2 for _ in range(B)]
    seed = 100
    for counts in ([70, 5, 0], [1, 1, 33], None, None, [40, 130, 2], None, [3, 0, 200], None, None):
        given = counts or [1] * B
        seed += 3
        k, v, q = (rand(sum(given), w * D, seed=seed + i) for i, w in enumerate((G, G, H)))
        cu = layer.append(k, v, counts)
        out, lse = zt.kv_cache.attn_rows(q, layer, H, G, D, cu_rows=cu, window=window, sinks=sinks, want_lse=True)
        at = 0
        for b, r in enumerate(given):
            held[b] = [torch.cat([x, y[at:at + r]]) for x, y in zip(held[b], (k, v))]
            if r:
                c = Case.__new__(Case)
                c.rows, c.past, c.H, c.G, c.D, c.window, c.sinks = [r], [len(held[b][0]) - r], H, G, D, window, sinks
                c.q, c.cu, c.keys = q[at:at + r], torch.tensor([0, r]), [held[b]]
                ref, ref_lse = c.reference(0)
                near(out[at:at + r], ref, (b, r))
                near(lse[at:at + r], ref_lse, (b, r))
            at += r
        layer.trim(window, sinks)
        if seed == 115:
            layer.release(1)
            held[1] = [x[:0] for x in held[1]]
    assert layer.len.tolist() == [len(x[0]) for x in held] == layer._len and int(layer.skipped) == 0
    with pytest.raises(zt.kv_cache.Full):
        layer.append(*(rand(600, G * D, seed=1) for _ in range(2)), [600, 0, 0])


@pytest.mark.parametrize("rows", [1, 20])
def test_captured_append_and_attention_replayed(zt, rows):
    """A loop of a graph's replays, in which every step appends behind the one before."""
    H, G, D, page, B = 8, 2, 128, 16, 3
    layer = zt.kv_cache.PagedLayer(60, page, G * D, B, 20)
    layer.reserve([200] * B)
    k, v, q = (torch.zeros(B * rows, w * D, device="cuda") for w in (G, G, H))
    cu = None if rows == 1 else torch.arange(0, (B + 1) * rows, rows, dtype=torch.int32, device="cuda")
    ws = zt.PagedWorkspace(B, B * rows, 20 * page, H, G, D)

    def step():
        zt.paged_append(layer.k, layer.v, layer.table, layer.len, k, v, cu_rows=cu)
        return zt.kv_cache.attn_rows(q, layer, H, G, D, cu_rows=cu, workspace=ws, want_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    layer.len.zero_()
    held = [[], []]
    for i in range(5):
        for x, y in zip((k, v, q), (rand(B * rows, w * D, seed=60 + 3 * i + j) for j, w in enumerate((G, G, H)))):
            x.copy_(y)
        held[0].append(k.clone().view(B, rows, -1)), held[1].append(v.clone().view(B, rows, -1))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            c = Case.__new__(Case)
            c.rows, c.past, c.H, c.G, c.D, c.window, c.sinks = [rows], [rows * i], H, G, D, 0, 0
            c.q, c.cu, c.keys = q[b * rows:(b + 1) * rows], torch.tensor([0, rows]), [[torch.cat([x[b] for x in y]) for y in held]]
            ref, ref_lse = c.reference(0)
            near(out[b * rows:(b + 1) * rows], ref, i)
            near(lse[b * rows:(b + 1) * rows], ref_lse, i)


def test_a_layer_decides_nothing_inside_a_capture(zt):
    """Its counts and pages are the host's, which a replay does not pass."""
    layer = zt.kv_cache.PagedLayer(8, 4, 64, 2, 4)
    layer.append(*(rand(2, 64, seed=5) for _ in range(2)))
    k, v, table, held = *(rand(2, 64, seed=6) for _ in range(2)), layer.table.clone(), (layer.free_pages(), list(layer._len))
    x = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        for call in (lambda: layer.append(k, v), lambda: layer.append(k, v, [1, 1]), lambda: layer.reserve([5, 5]), lambda: layer.release(0),
                     lambda: layer.trim(1)):
            with pytest.raises(zt.device.ConfigRefused, match="captured"):
                call()
    graph.replay()
    assert torch.equal(layer.table, table) and (layer.free_pages(), layer._len) == held and layer.len.tolist() == layer._len
    layer.append(k, v)
    assert layer.len.tolist() == [2, 2] == layer._len


def test_offsets_beyond_31_bits(zt):
    """Pages whose elements lie past 2^31 from the pool's begin."""
    H, G, D, page = 4, 2, 128, 256
    n_pages = 2**31 // (page * G * D) + 40
    free = torch.cuda.mem_get_info()[0]
    if free < 3 * n_pages * page * G * D * 4:
        pytest.skip("not enough device memory")
    kp, vp = (torch.empty(n_pages, page, G * D, device="cuda") for _ in range(2))
    for rows, past in ((30, 700), (1, 700)):
        c = Case([rows], [past], H, G, D, page, seed=2)
        ids = torch.tensor([n_pages - 1, 3, n_pages - 20, n_pages - 7], dtype=torch.int32, device="cuda")[:c.table.shape[1]]
        kp[ids.long()], vp[ids.long()] = c.k[c.table[0].long()], c.v[c.table[0].long()]
        c.k, c.v, c.table = kp, vp, ids[None].contiguous()
        c.check(*c.call(zt))
    n = torch.tensor([page - 1], dtype=torch.int32, device="cuda")
    new = rand(1, G * D, seed=8)
    zt.paged_append(kp, vp, ids[None].contiguous(), n, new, new)
    assert torch.equal(kp[n_pages - 1, page - 1], new[0]) and int(n) == page


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_table_too_long_to_convert_beforehand(zt, D):
    """Many rows over a table of a million places, nearly all without a page: the rows convert their own keys, and find the same."""
    c = Case([300, 500], [900, 40], 8, 2, D, 16, 100, 3, seed=23)
    ref = c.call(zt)
    room = zt.PagedWorkspace(2, c.N, c.table.shape[1] * 16, 8, 2, D).nbytes
    c.check(*ref)
    c.table = torch.nn.functional.pad(c.table, (0, 2**16 - c.table.shape[1]), value=-1)
    ws = zt.PagedWorkspace(2, c.N, 2**20, 8, 2, D)
    assert ws.nbytes > room
    out, lse = c.call(zt, workspace=ws)
    c.check(out, lse)
    near(out, ref[0].double(), "the two forms")


def test_numbers_at_the_edge_of_31_bits(zt):
    """Windows and sinks of any size, and a table whose capacity nearly fills 31 bits."""
    c = Case([40, 1], [100, 900], 8, 2, 64, 16, seed=24)
    for window, sinks in ((2**31 - 1, 0), (2**30 - 1, 2**31 - 1), (2**40, 2**40), (5, 2**31 - 1), (2**30 - 5, 3)):
        out, lse = zt.attention_paged(c.q, c.k, c.v, c.table, c.n_keys, 8, 2, 64, cu_rows=c.cu, window=window, sinks=sinks, want_lse=True)
        c.check(out, lse)
        s = Case([1, 1], [100, 900], 8, 2, 64, 16, seed=25)
        out, lse = zt.attention_paged(s.q, s.k, s.v, s.table, s.n_keys, 8, 2, 64, window=window, sinks=sinks, want_lse=True)
        s.check(out, lse)
    page = 2**24
    k = torch.zeros(1, 16, 128, device="cuda")  # (a pool of one page of 16 rows: no slot from 16 on is filled)
    table = torch.zeros(1, 127, dtype=torch.int32, device="cuda")
    n = torch.tensor([9], dtype=torch.int32, device="cuda")
    L = zt.lib.load()
    q, out = rand(9, 256, seed=1), torch.empty(9, 256, device="cuda")
    cu = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    ws = zt.PagedWorkspace(1, 9, 127 * page, 4, 2, 64)
    k.copy_(rand(1, 16, 128, seed=2))
    assert L.zt_attn_paged(q.data_ptr(), k.data_ptr(), k.data_ptr(), table.data_ptr(), n.data_ptr(), cu.data_ptr(), out.data_ptr(), None,
                           ws.buf.data_ptr(), ws.nbytes, 1, 9, 1, page, 127, 4, 2, 64, 3, 1, torch.cuda.current_stream().cuda_stream) == 0
    c = Case.__new__(Case)
    c.rows, c.past, c.H, c.G, c.D, c.window, c.sinks = [9], [0], 4, 2, 64, 3, 1
    c.q, c.cu, c.keys = q, torch.tensor([0, 9]), [[k[0, :9], k[0, :9]]]
    near(out, c.reference(0)[0], "one long page")


def test_on_another_stream_than_the_tensors_own(zt):
    c = Case([40, 3], [100, 900], 8, 2, 64, 16, seed=20)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out, lse = c.call(zt)
    s.synchronize()
    c.check(out, lse)
