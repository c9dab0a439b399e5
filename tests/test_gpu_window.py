"""Attention with a sliding window and sinks, forward and backward, against the formulas in 64 bits.

Tolerance: the stated bar of the attention paths, |got - ref| <= 1e-5 + 1e-4 |ref|, element-wise.  What the kernels owe it:
every f32 operand is two f16 pieces, so a product is off by 2^-21 of its factors' magnitudes at most, and sums of up to 600 such
terms of N(0, 1) inputs stay an order below the bar; the tests keep to such sizes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(*shape, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda")


def make(B, T, H, G, D, seed=0):
    q, dout = rand(B, T, H * D, seed=seed), rand(B, T, H * D, seed=seed + 1)
    return q, rand(B, T, G * D, seed=seed + 2), rand(B, T, G * D, seed=seed + 3), dout


def seen(T, window, sinks, device="cuda"):
    t, j = torch.arange(T, device=device)[:, None], torch.arange(T, device=device)[None, :]
    return (j <= t) & ((j > t - window) | (j < sinks)) if window else j <= t


def forward64(q, k, v, H, G, D, window, sinks):
    B, T = q.shape[:2]
    q, k, v = q.double().view(B, T, G, H // G, D), k.double().view(B, T, G, D), v.double().view(B, T, G, D)
    s = torch.einsum("btgrd,bsgd->bgrts", q, k) / math.sqrt(D)
    s = s.masked_fill(~seen(T, window, sinks, q.device), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    return torch.einsum("bgrts,bsgd->btgrd", p, v).reshape(B, T, H * D), lse.permute(0, 3, 1, 2).reshape(B, T, H), p


def backward64(q, k, v, dout, H, G, D, window, sinks):
    B, T = q.shape[:2]
    out, lse, p = forward64(q, k, v, H, G, D, window, sinks)
    q, k, v = q.double().view(B, T, G, H // G, D), k.double().view(B, T, G, D), v.double().view(B, T, G, D)
    g = dout.double().view(B, T, G, H // G, D)
    dp = torch.einsum("btgrd,bsgd->bgrts", g, v)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
    dq = torch.einsum("bgrts,bsgd->btgrd", ds, k).reshape(B, T, H * D)
    return out, lse, dq, torch.einsum("bgrts,btgrd->bsgd", ds, q).reshape(B, T, G * D), torch.einsum("bgrts,btgrd->bsgd", p, g).reshape(B, T, G * D)


def near(got, ref, what):
    err = (got.double() - ref).abs() - (1e-5 + 1e-4 * ref.abs())
    assert torch.isfinite(got).all() and err.max() <= 0, (what, float((got.double() - ref).abs().max()), float(err.max()))


SHAPES = [
    # (B, T, H, G, D, window, sinks): one row; a window of one; windows and sinks around the sequence's length
    (1, 1, 2, 1, 32, 1, 0), (2, 2, 4, 2, 64, 1, 1), (1, 33, 4, 4, 32, 1, 0), (1, 40, 4, 2, 32, 39, 0), (1, 40, 4, 2, 32, 40, 0),
    (1, 40, 4, 2, 32, 7, 40), (1, 40, 4, 2, 32, 1000, 1000), (2, 40, 4, 2, 32, 7, 39),
    # tile edges of rows, window and sinks
    (1, 127, 4, 2, 32, 64, 4), (1, 128, 4, 1, 64, 63, 0), (1, 129, 4, 2, 64, 65, 64), (2, 300, 8, 2, 64, 128, 65), (1, 513, 4, 4, 64, 127, 1),
    (1, 520, 3, 1, 64, 200, 130), (1, 600, 4, 2, 32, 33, 300),
    # other widths and groups
    (1, 260, 4, 2, 128, 100, 4), (2, 200, 6, 2, 96, 77, 3), (1, 190, 16, 4, 80, 50, 17), (1, 300, 5, 1, 100, 129, 5), (1, 140, 12, 4, 112, 31, 2),
    (1, 260, 4, 2, 256, 64, 4), (1, 200, 2, 2, 192, 90, 0), (2, 150, 4, 1, 160, 40, 33), (1, 330, 4, 2, 132, 131, 1), (1, 70, 32, 8, 128, 16, 2),
    # walks of many tiles: sinks' keys in several blocks, contractions in several pieces
    (1, 3000, 2, 1, 64, 100, 4), (2, 1400, 2, 1, 128, 60, 129), (1, 1500, 2, 1, 192, 300, 5), (1, 2300, 2, 1, 256, 100, 140),
    # widths that no tensor-core tile takes
    (1, 70, 4, 2, 34, 20, 3), (1, 50, 2, 1, 62, 33, 0), (1, 100, 4, 2, 36, 64, 1),
]


@pytest.mark.parametrize("B,T,H,G,D,window,sinks", SHAPES)
def test_forward_and_backward(zt, B, T, H, G, D, window, sinks):
    q, k, v, dout = make(B, T, H, G, D, seed=T + D)
    ref = backward64(q, k, v, dout, H, G, D, window, sinks)
    out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks, want_lse=True)
    alone = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks)
    ws = zt.BackwardWorkspace(B, T, H, G, D)
    ws.buf.fill_(255)
    got = zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks, workspace=ws)
    own = zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks)
    assert torch.equal(alone, out)
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got), ref):
        near(a, b, name)
    for a, b in zip(own, ref[2:]):
        near(a, b, "a workspace of its own")
    assert zt.lib.tc_status() == 0


def test_gradients_against_differences(zt):
    """(f(x + h e) - f(x - h e)) / 2h of f = sum(dout out) along random directions.  out is good to 1e-5 of its size, f to 1e-5 |dout|
    sqrt(n); with h = 0.05 the difference quotient's own error is h^2 times a third derivative of order |dout| |e|^3."""
    B, T, H, G, D, window, sinks = 1, 150, 4, 2, 64, 40, 3
    q, k, v, dout = make(B, T, H, G, D, seed=5)
    out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks, want_lse=True)
    grads = zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks)
    f = lambda *x: float((zt.attention_forward_window(*x, H, G, D, window, sinks=sinks).double() * dout.double()).sum())  # noqa: E731
    h = 0.05
    for i, g in enumerate(grads):
        e = rand(*g.shape, seed=70 + i)
        e /= e.norm()
        x = [q, k, v]
        up, down = ([y + s * h * e if j == i else y for j, y in enumerate(x)] for s in (1, -1))
        slope, want = (f(*up) - f(*down)) / (2 * h), float((g.double() * e.double()).sum())
        noise = 1e-6 * float(dout.norm()) / h  # f32 rounding of out, two evaluations
        assert abs(slope - want) <= noise + h * h * float(dout.abs().max()), (i, slope, want)


def test_a_window_that_leaves_nothing_out_is_the_plain_call(zt):
    B, T, H, G, D = 2, 200, 8, 2, 64
    q, k, v, dout = make(B, T, H, G, D)
    ref = backward64(q, k, v, dout, H, G, D, 0, 0)
    for window, sinks in ((0, 0), (T, 0), (2**40, 5), (3, T), (1, 2**35)):
        out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks, want_lse=True)
        grads = zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks)
        for a, b in zip((out, lse, *grads), ref):
            near(a, b, (window, sinks))


def test_python_refusals(zt):
    q, k, v, dout = make(1, 16, 4, 2, 32)
    E = zt.ops
    for bad in (dict(window=-1), dict(window=3, sinks=-1)):
        with pytest.raises(E.ConfigRefused):
            zt.attention_forward_window(q, k, v, 4, 2, 32, **bad)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_forward_window(q[0], k[0], v[0], 4, 2, 32, 3)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_forward_window(q, k[:, :8], v, 4, 2, 32, 3)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_forward_window(q.half(), k, v, 4, 2, 32, 3)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_forward_window(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, 4, 2, 32, 3)
    out, lse = zt.attention_forward_window(q, k, v, 4, 2, 32, 3, want_lse=True)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_backward_window(q, k, v, out, lse[:, :8], dout, 4, 2, 32, 3)
    with pytest.raises(E.DimensionMismatch):
        zt.attention_backward_window(q, k, v, out, lse, dout, 4, 2, 32, 3, workspace=zt.BackwardWorkspace(1, 17, 4, 2, 32))


@pytest.mark.parametrize("D", [64, 128])
def test_captured_and_replayed_on_new_inputs(zt, D):
    B, T, H, G, window, sinks = 1, 300, 4, 2, 90, 3
    q, k, v, dout = make(B, T, H, G, D)
    ws = zt.BackwardWorkspace(B, T, H, G, D)

    def step():
        out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks, want_lse=True)
        return (out, lse, *zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks, workspace=ws))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (21, 34):
        for x, y in zip((q, k, v, dout), make(B, T, H, G, D, seed=seed)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, backward64(q, k, v, dout, H, G, D, window, sinks)):
            near(a, b, seed)


def test_two_calls_at_once_on_two_streams(zt):
    """Nothing is shared: neither scratch nor workspace."""
    H, G, D, window, sinks = 8, 2, 64, 100, 4
    sides = [torch.cuda.Stream() for _ in range(2)]
    sets = [make(2, 700, H, G, D, seed=40 + i) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(sides):
            q, k, v, dout = sets[i]
            with torch.cuda.stream(s):
                out, lse = zt.attention_forward_window(q, k, v, H, G, D, window, sinks=sinks, want_lse=True)
                got[i].append((out, lse, *zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, window, sinks=sinks)))
    torch.cuda.synchronize()
    for i in range(2):
        ref = backward64(*sets[i], H, G, D, window, sinks)
        for one in got[i]:
            for a, b in zip(one, ref):
                near(a, b, i)
