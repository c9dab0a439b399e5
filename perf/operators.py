"""Attention over part of a prefix, as a training program and a serving program call it.

The rule of what is seen is one for all of them: the query at position p sees key j where j <= p and, with a window,
where j > p - window or j < sinks (the first tokens stay visible to every query).  Kinds of cases:

  train   attention_forward_window with its log-sum-exp, then attention_backward_window, over whole sequences
  prompt  attention_forward_window alone
  chunk   new tokens of several sequences enter a paged cache (paged_append), then attend over it (attention_paged)
  step    the same with one new token a sequence

Where `own` is false, run() computes the same from elementary torch operations in 32 bits, over the whole score matrix.
"""
import importlib
import math

import torch

own = False

#: (query heads, KV heads) of perf/cases.py
HEADS = ((4, 2), (8, 2), (12, 4), (16, 16), (32, 8))
#: its head widths, each as likely as its use
WIDTHS = (32, 64, 64, 96, 128, 128, 128, 192, 256)
PAGES = (8, 16, 16, 32, 50, 64, 128)
MAX_SCORES = 2 << 30       # entries of a case's whole score matrix
MAX_FLOPS = 4.5e11         # of its visible pairs
MAX_CACHE_BYTES = 4 << 30  # of its filled pages


def listed():
    return [
        # the reference's own training shape (context 256), with a window: launches and host work
        {"name": "train-t256-w64-d32", "kind": "train", "batch": 1, "t": 256, "heads": 4, "kv_heads": 2, "dim": 32,
         "window": 64, "sinks": 4},
        # a head width, a length and a window that no tile divides
        {"name": "train-t1000-w200-d80", "kind": "train", "batch": 4, "t": 1000, "heads": 16, "kv_heads": 4, "dim": 80,
         "window": 200, "sinks": 3},
        # a batch of middle-sized sequences
        {"name": "train-t2048-w512-d64", "kind": "train", "batch": 4, "t": 2048, "heads": 32, "kv_heads": 8, "dim": 64,
         "window": 512, "sinks": 4},
        # the widest heads, no sinks
        {"name": "train-t1024-w256-d256", "kind": "train", "batch": 2, "t": 1024, "heads": 16, "kv_heads": 4, "dim": 256,
         "window": 256, "sinks": 0},
        # long sequences of the benchmark's heads
        {"name": "train-t8192-w1024-d128", "kind": "train", "batch": 1, "t": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 1024, "sinks": 4},
        # a long prompt in a server, forward alone
        {"name": "prompt-t16384-w4096-d128", "kind": "prompt", "batch": 1, "t": 16384, "heads": 8, "kv_heads": 2, "dim": 128,
         "window": 4096, "sinks": 16},
        # a short follow-up of one conversation: 77 new tokens behind 923
        {"name": "chunk-r77-of-1000-d128", "kind": "chunk", "batch": 1, "rows": 77, "past": 923, "ragged": False, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0},
        # four long prompts a chunk at a time
        {"name": "chunk-r512-of-8192-d128", "kind": "chunk", "batch": 4, "rows": 512, "past": 7680, "ragged": False, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0},
        # what a scheduler packs together: sequences and chunks of all lengths, with a window
        {"name": "chunk-ragged-w2048-d64", "kind": "chunk", "batch": 32, "rows": 300, "past": 6000, "ragged": True, "page": 32,
         "heads": 16, "kv_heads": 16, "dim": 64, "window": 2048, "sinks": 4},
        # one user, one token: latency
        {"name": "step-b1-c1000-d128", "kind": "step", "batch": 1, "rows": 1, "past": 999, "ragged": False, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0},
        # the benchmark's decode batch over pages
        {"name": "step-b64-c8192-d128", "kind": "step", "batch": 64, "rows": 1, "past": 8191, "ragged": False, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0},
        # a large batch of unequal lengths, with a window and sinks
        {"name": "step-b256-ragged-w1024-d128", "kind": "step", "batch": 256, "rows": 1, "past": 3999, "ragged": True, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("train", "train", "train", "prompt", "chunk", "chunk", "chunk", "step", "step"))
    heads, kv_heads = rng.choice(HEADS)
    # one width in four is another multiple of four (36, 72, 100, 160, ...)
    dim = 4 * rng.randint(8, 64) if rng.random() < 0.25 else rng.choice(WIDTHS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if kind in ("train", "prompt"):
        case["batch"] = _log_int(rng, 1, 8)
        case["t"] = _log_int(rng, 16, 8192 if kind == "train" else 16384)
        case["window"] = _log_int(rng, 1, case["t"])
        case["sinks"] = rng.choice((0, 1, 4, 4, 16, 100))
    else:
        case["batch"] = _log_int(rng, 1, 64 if kind == "chunk" else 256)
        case["rows"] = 1 if kind == "step" else _log_int(rng, 2, 1024)
        case["past"] = _log_int(rng, 1, 16384) - 1
        case["ragged"] = rng.random() < 0.5
        case["page"] = rng.choice(PAGES)
        case["window"] = rng.choice((0, 0, _log_int(rng, 1, 4096)))
        case["sinks"] = rng.choice((0, 4, 16)) if case["window"] else 0
    while _scores(case) > MAX_SCORES or work(case)["flops"] > MAX_FLOPS or _cache_bytes(case) > MAX_CACHE_BYTES:
        if case["batch"] > 1:
            case["batch"] = case["batch"] * 2 // 3
        elif "t" in case:
            case["t"] = case["t"] * 4 // 5
            case["window"] = min(case["window"], case["t"])
        elif case["rows"] > 2:
            case["rows"] = case["rows"] * 2 // 3
        else:
            case["past"] = case["past"] * 2 // 3
    return case


def _lengths(case):
    """New rows and, with them, all keys of every sequence (before they are shuffled)."""
    B = case["batch"]
    if not case["ragged"]:
        return [case["rows"]] * B, [case["rows"] + case["past"]] * B
    rows = [max(1, case["rows"] * ((b * 7) % B + 1) // B) for b in range(B)]
    return rows, [r + case["past"] * ((b * 5 + 3) % B + 1) // B for b, r in enumerate(rows)]


def _scores(case):
    if "t" in case:
        return case["batch"] * case["heads"] * case["t"] ** 2
    rows, keys = _lengths(case)
    return case["batch"] * case["heads"] * max(rows) * max(keys)


def _cache_bytes(case):
    return 0 if "t" in case else 8 * sum(_lengths(case)[1]) * case["kv_heads"] * case["dim"]


def _pairs(first, last, window, sinks):
    """Visible (query, key) pairs of the queries at positions [first, last)."""
    if not window:
        return (last * (last + 1) - first * (first + 1)) // 2
    n = 0
    # up to `window` positions every key is seen; then the window and the sinks before it, which grow to `sinks`
    full = min(last, max(first, window))
    n += (full * (full + 1) - first * (first + 1)) // 2
    grown = min(last, max(full, window + sinks))  # at position p the window begins at p - window + 1
    n += sum(window + min(sinks, p - window + 1) for p in range(full, grown))
    return n + (last - grown) * (window + sinks)


def _keys_seen(first, last, window, sinks):
    """Keys that some query at positions [first, last) sees."""
    if not window:
        return last
    low = max(0, first - window + 1)
    return last - low + min(sinks, low)


def work(case):
    """Inputs that some query sees read once, outputs written once; the multiply-adds of the visible pairs."""
    H, G, D, w, s = (case[x] for x in ("heads", "kv_heads", "dim", "window", "sinks"))
    if "t" in case:
        B, T = case["batch"], case["t"]
        forward = 4 * B * H * D * _pairs(0, T, w, s)
        if case["kind"] == "prompt":
            return {"bytes": 4 * B * T * (2 * H * D + 2 * G * D + H), "flops": forward}
        return {"bytes": 4 * B * T * (4 * H * D + 4 * G * D + H), "flops": 3.5 * forward}
    n = flops = moved = 0
    for r, keys in zip(*_lengths(case)):
        n += r
        flops += 4 * H * D * _pairs(keys - r, keys, w, s)
        moved += 4 * 2 * G * D * _keys_seen(keys - r, keys, w, s)
    return {"bytes": moved + 4 * n * (2 * H * D + H + 4 * G * D), "flops": flops}


def _normal(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return lambda *shape: torch.randn(shape, dtype=torch.float32, device="cuda", generator=gen)


def prepare(case, seed):
    normal = _normal(seed)
    B, H, G, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if "t" in case:
        T = case["t"]
        s.update(q=normal(B, T, H * D), k=normal(B, T, G * D), v=normal(B, T, G * D))
        if case["kind"] == "train":
            s["dout"] = normal(B, T, H * D)
        return s
    host = torch.Generator()
    host.manual_seed(seed)
    order = torch.randperm(B, generator=host).tolist()
    rows, keys = ([x[i] for i in order] for x in _lengths(case))
    ps = case["page"]
    used = [-(-x // ps) for x in keys]
    n_pages, most = sum(used) + 3, max(used)
    # pages lie in the pool in no order; the table's places without a page hold -1
    shuffled = torch.randperm(n_pages, generator=host, dtype=torch.int32)
    table = torch.full((B, most), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = shuffled[at:at + u]
        at += u
    cu = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    N = int(cu[-1])
    s.update(q=normal(N, H * D), k_new=normal(N, G * D), v_new=normal(N, G * D), k_pages=normal(n_pages, ps, G * D),
             v_pages=normal(n_pages, ps, G * D), table=table.cuda(), cu_rows=cu.cuda(),
             filled=torch.tensor([k - r for k, r in zip(keys, rows)], dtype=torch.int32).cuda())
    s["n_keys"] = s["filled"].clone()
    return s


def _zt():
    return importlib.import_module("z-transformer_b200")


def run(s):
    if "q" in s and "table" in s:
        s["n_keys"].copy_(s["filled"])  # back to the cache before these tokens: they are written again
        return _run_paged_own(s) if own else _run_paged_plain(s)
    return _run_whole_own(s) if own else _run_whole_plain(s)


def _run_whole_own(s):
    zt, c = _zt(), s["case"]
    H, G, D, w, n = c["heads"], c["kv_heads"], c["dim"], c["window"], c["sinks"]
    q, k, v = s["q"], s["k"], s["v"]
    out, lse = zt.attention_forward_window(q, k, v, H, G, D, w, sinks=n, want_lse=True)
    if c["kind"] == "prompt":
        return {"out": out, "lse": lse}
    if "workspace" not in s:
        s["workspace"] = zt.BackwardWorkspace(c["batch"], c["t"], H, G, D)  # lives as long as the training does
    dq, dk, dv = zt.attention_backward_window(q, k, v, out, lse, s["dout"], H, G, D, w, sinks=n, workspace=s["workspace"])
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _run_paged_own(s):
    zt, c = _zt(), s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    cu = None if c["kind"] == "step" else s["cu_rows"]
    if "workspace" not in s:
        s["workspace"] = zt.PagedWorkspace(c["batch"], s["q"].shape[0], s["table"].shape[1] * c["page"], H, G, D)
    zt.paged_append(s["k_pages"], s["v_pages"], s["table"], s["n_keys"], s["k_new"], s["v_new"], cu_rows=cu)
    out, lse = zt.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["n_keys"], H, G, D, cu_rows=cu,
                                  window=c["window"], sinks=c["sinks"], workspace=s["workspace"], want_lse=True)
    return {"out": out, "lse": lse, "n_keys": s["n_keys"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _seen(pos, key, window, sinks):
    seen = key <= pos
    return seen & ((key > pos - window) | (key < sinks)) if window else seen


def _run_whole_plain(s):
    c = s["case"]
    B, T, H, G, D = c["batch"], c["t"], c["heads"], c["kv_heads"], c["dim"]
    R, scale = H // G, 1.0 / math.sqrt(D)
    rows = lambda x: x.view(B, T, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * T, D)  # noqa: E731
    back = lambda x: x.view(B, G, R, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H * D)  # noqa: E731
    q, k, v = rows(s["q"]), s["k"].view(B, T, G, D).transpose(1, 2), s["v"].view(B, T, G, D).transpose(1, 2)
    at = torch.arange(T, device=q.device)
    seen = _seen(at[:, None], at[None, :], c["window"], c["sinks"])
    p = (q @ k.transpose(2, 3)).mul_(scale).view(B, G, R, T, T).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    p = p.div_(den).view(B, G, R * T, T)
    lse = (top + den.log()).view(B, G, R, T).permute(0, 3, 1, 2).reshape(B, T, H)
    out = p @ v
    if c["kind"] == "prompt":
        return {"out": back(out), "lse": lse}
    g = rows(s["dout"])
    delta = (g * out).sum(-1, keepdim=True)
    dv = p.transpose(2, 3) @ g
    ds = (g @ v.transpose(2, 3)).sub_(delta).mul_(p)
    dq = (ds @ k).mul_(scale)
    dk = (ds.transpose(2, 3) @ q).mul_(scale)
    flat = lambda x: x.transpose(1, 2).reshape(B, T, G * D)  # noqa: E731
    return {"out": back(out), "lse": lse, "dq": back(dq), "dk": flat(dk), "dv": flat(dv)}


def _run_paged_plain(s):
    c = s["case"]
    B, H, G, D, ps = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    R, cu, table, n_keys = H // G, s["cu_rows"].long(), s["table"].long(), s["n_keys"]
    rows = cu[1:] - cu[:-1]
    N, most = s["q"].shape[0], max(_lengths(c)[0])
    # the new rows into their places
    at = torch.arange(N, device=cu.device)
    seq = (at[:, None] >= cu[None, 1:]).sum(1)
    slot = n_keys.long()[seq] + at - cu[seq]
    page = table[seq, slot // ps]
    s["k_pages"][page, slot % ps] = s["k_new"]
    s["v_pages"][page, slot % ps] = s["v_new"]
    n_keys += rows.int()
    # every sequence's keys in a row, and its queries padded to the longest chunk
    keys = lambda x: x[table.clamp(min=0)].view(B, -1, G, D).transpose(1, 2)  # noqa: E731
    k, v = keys(s["k_pages"]), keys(s["v_pages"])
    i = torch.arange(most, device=cu.device)
    here = i[None, :] < rows[:, None]
    q = s["q"][(cu[:-1, None] + i[None, :]).clamp(max=N - 1)].view(B, most, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * most, D)
    pos = (n_keys.long() - rows)[:, None] + i[None, :]
    seen = _seen(pos[:, :, None], torch.arange(k.shape[2], device=cu.device)[None, None, :], c["window"], c["sinks"])
    p = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(B, G, R, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    out = (p.div_(den).view(B, G, R * most, -1) @ v).view(B, G, R, most, D).permute(0, 3, 1, 2, 4)
    lse = (top + den.log()).view(B, G, R, most).permute(0, 3, 1, 2)
    return {"out": out[here].reshape(N, H * D), "lse": lse[here].reshape(N, H), "n_keys": n_keys, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _head_64(q, k, v, pos, window, sinks, dout=None):
    """One KV head of one sequence in 64 bits: q, dout [rows, heads of the group, D] at positions pos, k and v [keys, D]."""
    D = q.shape[-1]
    j = torch.arange(k.shape[0], device=k.device)
    hidden = j[None, :] > pos[:, None]
    if window > 0:
        hidden |= (j[None, :] <= pos[:, None] - window) & (j[None, :] >= sinks)
    x = torch.einsum("rhd,kd->rhk", q, k) / D ** 0.5
    x[hidden[:, None, :].expand_as(x)] = -math.inf
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[:, :, None])
    del x
    out = torch.einsum("rhk,kd->rhd", p, v)
    if dout is None:
        return out, lse
    dv = torch.einsum("rhk,rhd->kd", p, dout)
    dp = torch.einsum("rhd,kd->rhk", dout, v)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / D ** 0.5
    return out, lse, torch.einsum("rhk,kd->rhd", ds, k), torch.einsum("rhk,rhd->kd", ds, q), dv


def exact(case, seed):
    s = prepare(case, seed)
    B, H, G, D, w, n = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "window", "sinks"))
    R = H // G
    if "t" in case:
        T = case["t"]
        pos = torch.arange(T, device="cuda")
        wide = {x: s[x].view(B, T, -1, D) for x in ("q", "k", "v", "dout") if x in s}
        names = ("out", "lse") if case["kind"] == "prompt" else ("out", "lse", "dq", "dk", "dv")
        got = {x: torch.zeros((B, T, {"lse": H, "dk": G * D, "dv": G * D}.get(x, H * D)), dtype=torch.float64, device="cuda") for x in names}
        for b in range(B):
            for g in range(G):
                hs = slice(g * R, (g + 1) * R)
                one = _head_64(wide["q"][b, :, hs].double(), wide["k"][b, :, g].double(), wide["v"][b, :, g].double(), pos, w, n,
                               wide["dout"][b, :, hs].double() if "dout" in wide else None)
                for x, y in zip(names, one):
                    per = {"lse": R, "dk": D, "dv": D}.get(x, R * D)
                    got[x][b, :, g * per:(g + 1) * per] = y.reshape(T, per)
        return got
    ps, cu, table, filled = case["page"], s["cu_rows"].tolist(), s["table"].tolist(), s["filled"].tolist()
    N = cu[-1]
    out = torch.zeros((N, G, R, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((N, G, R), dtype=torch.float64, device="cuda")
    for b in range(B):
        r0, r1, before = cu[b], cu[b + 1], filled[b]
        total = before + r1 - r0
        at = torch.arange(before, total, device="cuda")
        pages = torch.tensor(table[b][:-(-total // ps)], device="cuda")
        for x in "kv":
            s[x + "_pages"][pages[at // ps], at % ps] = s[x + "_new"][r0:r1]
        k, v = (s[x + "_pages"][pages].view(-1, G, D)[:total] for x in "kv")
        q = s["q"][r0:r1].view(-1, G, R, D)
        for g in range(G):
            out[r0:r1, g], lse[r0:r1, g] = _head_64(q[:, g].double(), k[:, g].double(), v[:, g].double(), at, w, n)
    lens = s["filled"] + s["cu_rows"][1:] - s["cu_rows"][:-1]
    return {"out": out.view(N, H * D), "lse": lse.view(N, H), "n_keys": lens, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
