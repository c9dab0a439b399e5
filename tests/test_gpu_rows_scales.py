"""Keys and values whose magnitude changes from tile to tile (as the first tokens' often does) or inside one, against the formulas in 64 bits, in both
forms of the rows' kernel: a tile that the row tile converts itself takes the scale that the tile before would have had, where that will do.

Tolerance, of a (row, head)'s columns as a vector: 5e-6 of the norm of sum p |v|.  S, by its 8 to 40 additions to a growing sum, is off by 1.8e-6 of itself
at most (2^-24 * 2/3 each, and the pieces' 2^-23), and stands at two where weights count: 3.6e-6 of a weight.  The pieces of v keep 22 bits, 2.4e-7.
P V: 12 additions, 5e-7.  What is added to that: a value's lo piece is a multiple of 2^-24 where the tile's largest value is 2^12 at least (2^4 where the
scale is the tile's before), so it is off by 2^-25 / 2^12 = 2^-37 (2^-29) of the largest value of its tile, 128 keys at most; the weights' sum is one."""
import math

import pytest
import torch
from test_gpu_paged import Case
from test_gpu_window import make, seen

pytestmark = pytest.mark.gpu


def factors(n, pattern):
    j = torch.arange(n, device="cuda")
    tile = j // 64
    f = torch.ones(n, device="cuda")
    if pattern == "sinks":  # the first four tokens, a hundred thousand times the others
        f[:4] = 1e5
    elif pattern == "small sinks":
        f[:4] = 1e-5
    elif pattern == "tiles":  # each way, by factors that the carried scale bears and by others
        f = torch.tensor([1.0, 1e3, 1e-3, 1e6, 1.0, 4e-5, 8.0, 3e4, 1e-2], device="cuda")[tile % 9]
    elif pattern == "halves":  # changes that do not fall on tiles
        f = torch.tensor([1.0, 2e4, 3e-4, 1.0, 1e-6], device="cuda")[(j + 41) // 100 % 5]
    elif pattern == "a row":  # one key of every tile but the first
        f[75::64] = 1e4
    elif pattern == "zeros":  # first parts and whole tiles of zeros, then large and small
        f = torch.where((tile % 3 == 1) | (j % 64 < 16), 0.0, torch.where(tile % 2 == 0, 1e4, 1e-4))
    elif pattern == "far":
        f = torch.tensor([1e-30, 1e30, 1.0, 1e-18], device="cuda")[tile % 4]
    return f


PATTERNS = ["sinks", "small sinks", "tiles", "halves", "a row", "zeros", "far"]


def close(out, lse, q, k, v, hidden, what, beside=2.0**-29, tile=128):
    """q [t, H, D], k, v [s, G, D] as the kernel had them; `beside`: of the largest value in the tiles that the row sees."""
    t, H, D = q.shape
    G = k.shape[1]
    s = torch.einsum("tgrd,sgd->grts", q.double().view(t, G, H // G, D), k.double()) / math.sqrt(D)
    s = s.masked_fill(hidden, -math.inf)
    want = torch.logsumexp(s, -1)
    p = torch.exp(s - want[..., None])
    back = lambda x: x.permute(2, 0, 1, 3).reshape(t, H, D)  # noqa: E731
    ref, size = back(torch.einsum("grts,sgd->grtd", p, v.double())), back(torch.einsum("grts,sgd->grtd", p, v.double().abs()))
    n = -(-k.shape[0] // tile)
    most = torch.nn.functional.pad(v.abs(), (0, 0, 0, 0, 0, n * tile - v.shape[0])).view(n, tile, G, D).amax((1, 3))  # [tile, KV head]
    visits = torch.nn.functional.pad(~hidden, (0, n * tile - v.shape[0])).view(t, n, tile).any(-1)
    most = (visits[:, :, None] * most[None]).amax(1).repeat_interleave(H // G, 1)  # [t, H]
    off = (out.view(t, H, D).double() - ref).norm(dim=-1) - beside * math.sqrt(D) * most
    off = off / size.norm(dim=-1).clamp(min=1e-300)
    assert torch.isfinite(out).all() and float(off.max()) <= 5e-6, (what, float(off.max()), int(off.argmax()) // H)
    got, want = lse.view(t, H).double(), want.permute(2, 0, 1).reshape(t, H)
    assert ((got - want).abs() <= 1e-5 + 1e-6 * want.abs()).all(), (what, float((got - want).abs().max()))


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (8, 2, 128), (8, 2, 256), (4, 2, 80)])
@pytest.mark.parametrize("rows,window", [(3, 0), (40, 0), (40, 90), (300, 0), (300, 90)])
def test_over_pages(zt, pattern, H, G, D, rows, window):
    past, sinks = 650, 4 if window else 0
    c = Case([rows], [past], H, G, D, 16, 0, 0, seed=rows + D)
    n = rows + past
    ids, j = c.table[0].long()[torch.arange(n, device="cuda") // 16], torch.arange(n, device="cuda") % 16
    pos = torch.arange(past, n, device="cuda")[:, None]
    at = torch.arange(n, device="cuda")[None, :]
    hidden = at > pos if not window else (at > pos) | ((at <= pos - window) & (at >= sinks))
    f = factors(n, pattern)[:, None]
    k0, v0 = c.keys[0]
    # values; then keys, with q so small that the largest give scores of one
    for what, kf, vf, qf in (("v", torch.ones_like(f), f, 1.0), ("k", f, torch.ones_like(f), 1.0 / float(f.max()))):
        k, v, q = k0 * kf, v0 * vf, c.q * qf
        c.k[ids, j], c.v[ids, j] = k, v
        out, lse = zt.attention_paged(q, c.k, c.v, c.table, c.n_keys, H, G, D, cu_rows=c.cu, window=window, sinks=sinks, want_lse=True)
        close(out, lse, q.view(rows, H, D), k.view(n, G, D), v.view(n, G, D), hidden, what)
    assert zt.lib.tc_status() == 0


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("T,H,G,D,window", [(700, 4, 2, 64, 90), (700, 8, 2, 64, 300), (700, 4, 4, 128, 40), (700, 8, 2, 128, 300), (700, 4, 2, 256, 90)])
def test_whole_sequences(zt, pattern, T, H, G, D, window):
    q0, k0, v0, _ = make(1, T, H, G, D, seed=T + D)
    f = factors(T, pattern)[:, None]
    hidden = ~seen(T, window, 4)
    for what, k, v, q in (("v", k0, v0 * f, q0), ("k", k0 * f, v0, q0 / float(f.max()))):
        out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=4, want_lse=True)
        close(out[0], lse[0], q.view(T, H, D), k.view(T, G, D), v.view(T, G, D), hidden, what)
    assert zt.lib.tc_status() == 0


@pytest.mark.parametrize("D,past,rows,tile,window", [(64, 672, 64, 128, 60), (128, 724, 44, 64, 30), (256, 677, 27, 32, 12)])
def test_small_values_beside_others_in_a_tile_much_smaller_than_the_one_before(zt, D, past, rows, tile, window):
    """Tiles fall by 2^14 and rise again; of a small one the first quarter is a thousand times larger than what follows.  Rows that see only this have the
    tile's own scale for it, 2^-37 of the tile's largest."""
    H, G = 4, 2
    c = Case([rows], [past], H, G, D, 16, 0, 0, seed=D)
    n = rows + past
    ids, j = c.table[0].long()[torch.arange(n, device="cuda") // 16], torch.arange(n, device="cuda")
    small = j // tile % 2 == 1
    f = torch.where(small, torch.where(j % tile < tile // 4, 2.0**-14, 2.0**-14 / 1000), 1.0)[:, None]
    k, v = c.keys[0][0], c.keys[0][1] * f
    c.k[ids, j % 16], c.v[ids, j % 16] = k, v
    pos = torch.arange(past, n, device="cuda")[:, None]
    hidden = (j > pos) | (j <= pos - window)
    out, lse = zt.attention_paged(c.q, c.k, c.v, c.table, c.n_keys, H, G, D, cu_rows=c.cu, window=window, want_lse=True)
    close(out, lse, c.q.view(rows, H, D), k.view(n, G, D), v.view(n, G, D), hidden, "v", 2.0**-37, tile)
    assert ((~hidden) & (f[:, 0] > 1e-6)).any(1).logical_not().any()  # (some see only the smallest)
