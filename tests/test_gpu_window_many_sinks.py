"""Windows with tens of thousands of sinks: their backward is more blocks than a grid takes along y.  Tolerance: that of test_gpu_window.py; a
weight is about one over the keys that are seen, so sums over more queries than there are smaller for it."""
import math

import pytest
import torch
from test_gpu_window import make, near

pytestmark = pytest.mark.gpu


def backward64(q, k, v, dout, H, D, window, sinks, step=2048):
    """One sequence of one KV head in 64 bits, some queries at a time, over the keys that these see."""
    T = q.shape[1]
    q, dout = (x[0].double().view(T, H, D) for x in (q, dout))
    k, v = k[0].double(), v[0].double()
    out, lse, dq = torch.empty_like(q), torch.empty(T, H, dtype=torch.float64, device="cuda"), torch.empty_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for t0 in range(0, T, step):
        t1 = min(T, t0 + step)
        first = min(sinks, t1)
        j = torch.cat([torch.arange(first, device="cuda"), torch.arange(max(first, t0 - window + 1), t1, device="cuda")])
        t = torch.arange(t0, t1, device="cuda")[:, None]
        hidden = (j > t) | ((j <= t - window) & (j >= sinks))
        for h in range(H):
            s = (q[t0:t1, h] @ k[j].T / math.sqrt(D)).masked_fill_(hidden, -math.inf)
            lse[t0:t1, h] = torch.logsumexp(s, -1)
            p = s.sub_(lse[t0:t1, h, None]).exp_()
            g = dout[t0:t1, h]
            out[t0:t1, h] = p @ v[j]
            dv.index_add_(0, j, p.T @ g)
            ds = (g @ v[j].T).sub_((g * out[t0:t1, h]).sum(-1, keepdim=True)).mul_(p).div_(math.sqrt(D))
            dq[t0:t1, h] = ds @ k[j]
            dk.index_add_(0, j, ds.T @ q[t0:t1, h])
    return out.view(1, T, H * D), lse[None], dq.view(1, T, H * D), dk[None], dv[None]


@pytest.mark.parametrize("T,H,D,window,sinks", [(131072, 2, 128, 64, 32768), (131072, 1, 64, 64, 32768), (65536, 1, 80, 1, 65535)])
def test_forward_and_backward(zt, T, H, D, window, sinks):
    q, k, v, dout = make(1, T, H, 1, D, seed=T + D)
    out, lse = zt.attention_forward_window(q, k, v, H, 1, D, window, sinks=sinks, want_lse=True)
    ws = zt.BackwardWorkspace(1, T, H, 1, D)
    got = zt.attention_backward_window(q, k, v, out, lse, dout, H, 1, D, window, sinks=sinks, workspace=ws)
    torch.cuda.synchronize()
    ref = backward64(q, k, v, dout, H, D, window, sinks)
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got), ref):
        near(a, b, name)
    assert zt.lib.tc_status() == 0
