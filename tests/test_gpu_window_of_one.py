"""A window of one key without sinks: a query sees itself alone, so out is v, dv sums dout over the group's heads, and dq and dk are zero, not the
rounding of dP and delta."""
import math

import pytest
import torch
from test_gpu_window import backward64, make, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H,G,D", [(1, 1, 2, 1, 64), (2, 50, 4, 2, 32), (1, 300, 8, 2, 64), (2, 260, 6, 2, 96), (1, 200, 4, 2, 128), (1, 300, 4, 2, 256), (1, 70, 4, 2, 34), (1, 1100, 2, 1, 192)])
@pytest.mark.parametrize("path", [0, 1, 8])
def test_gradients_are_zero(zt, B, T, H, G, D, path):
    q, k, v, dout = make(B, T, H, G, D, seed=T + D)
    old = zt.lib.load().zt_attn_set_path(path)
    try:
        out, lse = zt.attention_forward_window(q, k, v, H, G, D, 1, want_lse=True)
        got = zt.attention_backward_window(q, k, v, out, lse, dout, H, G, D, 1)
        two = zt.attention_forward_window(q, k, v, H, G, D, 1, sinks=1, want_lse=True)
        both = zt.attention_backward_window(q, k, v, *two, dout, H, G, D, 1, sinks=1)
    finally:
        zt.lib.load().zt_attn_set_path(old)
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got), backward64(q, k, v, dout, H, G, D, 1, 0)):
        near(a, b, name)
    assert (got[0] == 0).all() and (got[1] == 0).all()
    # With a sink the queries behind it see two keys.  Its gradients are sums of T terms: an f32 addition is off by 2^-25 of the sum at most, with
    # either sign, 2^-25 / sqrt(3) on average; four times that of sqrt(T) additions is sqrt(T) 2^-24 * 1.2 of the largest sum.
    for a, b in zip((*two, *both), backward64(q, k, v, dout, H, G, D, 1, 1)):
        err = (a.double() - b).abs() - (1e-5 + 1e-4 * b.abs() + math.sqrt(T) * 2.0**-24 * 1.2 * b.abs().max())
        assert float(err.max()) <= 0, float(err.max())
    assert zt.lib.tc_saturated() == 0
