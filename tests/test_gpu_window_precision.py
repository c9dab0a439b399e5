"""How exact windows' outputs are, as the norm of the error over the norm of the result.  The tensor core adds with truncation: an addition to a
sum that has grown loses half a step of 2^-23 on average, 2^-24 of the sum, which on its way is two thirds of what it becomes.  The small terms
of the f16 pieces cost nothing while they come first."""
import math

import pytest
import torch
from test_gpu_paged import Case
from test_gpu_window import backward64, make, seen

pytestmark = pytest.mark.gpu


def errors(zt, B, T, H, G, D, window, sinks):
    q, k, v, dout = make(B, T, H, G, D, seed=T + D)
    ref = backward64(q, k, v, dout, H, G, D, window, sinks)
    out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks, want_lse=True)
    got = zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks)
    return {n: float((a.double() - b).norm() / b.norm()) for n, a, b in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got), ref)}


@pytest.mark.parametrize("B,T,H,G,D,window,sinks", [(4, 1000, 16, 4, 80, 200, 3), (1, 1000, 16, 4, 128, 300, 4), (1, 1000, 16, 4, 128, 1000, 0), (1, 2000, 8, 2, 128, 600, 4)])
def test_heads_of_65_to_128_columns(zt, B, T, H, G, D, window, sinks):
    """S: eight additions to a growing sum, 8 * 2^-24 * 2/3 = 3.2e-7 of S, which is near one, and so of a weight; out sums weighted values whose errors
    are partly their common bias, which the softmax takes out: 4.2e-7 with a third for P's pieces and P V.  (With the small terms of the second half behind the
    hi ones of the first it is sixteen additions, and 4.7e-7 to 5.5e-7 were measured.)  dv: 128 rows between two flushes, in two steps: 4 + 12 additions,
    16 * 2^-24 * 2/3 = 6.4e-7.  Its weights' error is 3.2e-7 of S less the row's mean under P; where they count, by their squares, a score of variance one
    stands at two and the mean at one: sqrt(1 + 1) * 3.2e-7 = 4.5e-7; pieces, 2^-23: 1.2e-7.  Together 1.21e-6 at most."""
    e = errors(zt, B, T, H, G, D, window, sinks)
    assert e["out"] <= 4.2e-7 and e["dv"] <= 1.25e-6, e


@pytest.mark.parametrize("B,T,H,G,D,window,sinks", [(1, 2000, 4, 2, 192, 900, 4), (1, 3000, 4, 2, 256, 1500, 4), (2, 1024, 16, 4, 256, 256, 0), (1, 700, 4, 1, 160, 300, 5)])
def test_heads_above_128_columns(zt, B, T, H, G, D, window, sinks):
    """dq, dk and dv: 128 contraction rows an accumulator in two steps, 4 + 12 additions to a growing sum: 16 * 2^-24 * 2/3 = 6.4e-7.  S and dP: as many
    additions as the head has sixteens of columns, n * 2^-24 * 2/3 of each, 6.4e-7 at 256; of S what a weight notices is sqrt(2) times that (see above).  In
    quadrature at 256: dq and dk 1.28e-6, dv 1.11e-6.  out: S, and 4.8e-7 (see test_rows_over_pages).  (With the small terms of 64 columns behind the
    hi ones of the last, and one accumulator for 1024 rows, dk's 2.5e-6 to 6.1e-6 and out's 6.1e-7 to 1.0e-6 were measured.)"""
    e = errors(zt, B, T, H, G, D, window, sinks)
    sums, s, dp = 6.4e-7, math.sqrt(2) * D / 16 * 2.0**-24 * 2 / 3, D / 16 * 2.0**-24 * 2 / 3
    assert e["dk"] <= math.hypot(sums, s, dp) and e["dq"] <= math.hypot(sums, s, dp) and e["dv"] <= math.hypot(sums, s), e
    assert e["out"] <= math.hypot(s, 4.8e-7), e


@pytest.mark.parametrize("H,G,D", [(8, 2, 256), (8, 2, 192), (16, 4, 128), (8, 2, 160)])
@pytest.mark.parametrize("rows", [25, 300])
def test_rows_over_pages(zt, H, G, D, rows):
    """S: as many additions to a growing sum as the head has sixteens of columns, n * 2^-24 * 2/3 of S.  What out notices of it is S less the row's mean
    under P, where weights count by their squares: sqrt(2) of that (see above), 9.0e-7 at 256.  In quadrature with 4.8e-7: P V, four additions a tile, 1.6e-7;
    P's pieces 1.2e-7; the tiles' sums in registers 1e-7; the exponent, a number near eight rounded at 2^-24 of itself, 4.2e-7.  (With the small terms of
    64 columns behind the hi ones of the last 8.4e-7 at 160, 9.1e-7 at 192 and 1.2e-6 at 256 were measured.)"""
    c = Case([rows], [1500], H, G, D, 16, seed=D)
    out, _ = c.call(zt)
    ref = c.reference(0)[0]
    bound = math.hypot(math.sqrt(2) * D / 16 * 2.0**-24 * 2 / 3, 4.8e-7)
    assert float((out.double() - ref).norm() / ref.norm()) <= bound


@pytest.mark.parametrize("B,T,H,G,D,window,sinks", [(4, 1000, 16, 4, 80, 200, 3), (1, 1000, 16, 4, 128, 300, 4), (1, 700, 8, 2, 112, 150, 0), (2, 500, 4, 4, 128, 400, 2), (1, 1000, 16, 4, 192, 300, 4), (2, 1024, 16, 4, 256, 256, 0)])
def test_gradients_beside_a_plain_form_in_32_bits(zt, B, T, H, G, D, window, sinks):
    """At most half as much again as what sums in 32 bits leave, or 1e-6."""
    q, k, v, dout = make(B, T, H, G, D, seed=T + D)
    ref = backward64(q, k, v, dout, H, G, D, window, sinks)
    R, scale = H // G, 1.0 / math.sqrt(D)
    qs, gs = (x.view(B, T, G, R, D) for x in (q, dout))
    ks, vs = (x.view(B, T, G, D) for x in (k, v))
    assert not torch.backends.cuda.matmul.allow_tf32
    s = (torch.einsum("btgrd,bsgd->bgrts", qs, ks) * scale).masked_fill(~seen(T, window, sinks), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    delta = (gs * torch.einsum("bgrts,bsgd->btgrd", p, vs)).sum(-1).permute(0, 2, 3, 1)[..., None]
    ds = p * (torch.einsum("btgrd,bsgd->bgrts", gs, vs) - delta)
    plain = {"dq": (torch.einsum("bgrts,bsgd->btgrd", ds, ks) * scale).reshape(B, T, H * D), "dk": (torch.einsum("bgrts,btgrd->bsgd", ds, qs) * scale).reshape(B, T, G * D),
             "dv": torch.einsum("bgrts,btgrd->bsgd", p, gs).reshape(B, T, G * D)}
    e = errors(zt, B, T, H, G, D, window, sinks)
    for name, want in zip(("dq", "dk", "dv"), ref[2:]):
        theirs = float((plain[name].double() - want).norm() / want.norm())
        assert e[name] <= max(1e-6, 1.5 * theirs), (name, e[name], theirs)
