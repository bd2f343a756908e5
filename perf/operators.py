"""The operators around attention whose speed and results are measured, as training and serving
programs call them:

  norm_rope   `tattn.qk_norm_rope`: root-mean-square norm of every query and key head and the
              position rotation, with the gradients of the inputs and of both weights
  window      `tattn.window_attention`: causal attention that sees the last `window` keys and the
              first `sinks` ones, grouped heads; training, prompts, and one token over a cache
  tables      `tattn.page_tables`: pages for the tokens that requests add, and the tokens' slots
  write       `tattn.cache4_write` and `tattn.cache4_read`: tokens into the pages of a cache held
              in 4 bits, and the values it then holds for them
  attend      `tattn.cache4_attention`: one token per request over that cache

The cache holds blocks of 32 values along the head as 4-bit codes (sign, two exponent bits, one
mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times a power of two, the smallest one at which the block's
largest magnitude rounds to 6 or less. Codes lie in [pages, kv heads, 2, page size, d / 2] bytes, an
even index in the low half, exponents (biased by 127) in [pages, kv heads, 2, page size, d / 32].
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


@functools.lru_cache(maxsize=None)
def _tattn():
    pkg = str(Path(__file__).resolve().parent.parent / "triton-attn_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tattn

    return tattn


# ---- cases ---------------------------------------------------------------------------------------

def _norm_rope(name, z, h, hk, n, d, dtype, train, layout="tokens", interleaved=False):
    return {"name": name, "op": "norm_rope", "z": z, "h": h, "hk": hk, "n": n, "d": d, "dtype": dtype,
            "train": train, "layout": layout, "interleaved": interleaved}


def _window(name, z, h, hk, n, s, d, window, sinks, dtype, train, lens=False, layout="heads"):
    return {"name": name, "op": "window", "z": z, "h": h, "hk": hk, "n": n, "s": s, "d": d, "window": window,
            "sinks": sinks, "dtype": dtype, "train": train, "lens": lens, "layout": layout}


def _tables(name, requests, longest, new, page):
    return {"name": name, "op": "tables", "requests": requests, "longest": longest, "new": new, "page": page}


def _write(name, tokens, hk, d, page, dtype):
    return {"name": name, "op": "write", "tokens": tokens, "hk": hk, "d": d, "page": page, "dtype": dtype}


def _attend(name, requests, longest, h, hk, d, page, window, sinks, dtype):
    return {"name": name, "op": "attend", "requests": requests, "longest": longest, "h": h, "hk": hk, "d": d,
            "page": page, "window": window, "sinks": sinks, "dtype": dtype}


def listed():
    return [
        # One decoding step of 32 sequences: every launch is latency.
        _norm_rope("norm_rope_one_token", 32, 16, 4, 1, 128, "bf16", False),
        # A training step's queries and keys, grouped heads, as the projection leaves them.
        _norm_rope("norm_rope_train", 4, 32, 8, 4096, 128, "bf16", True),
        # The benchmark's middle length trained with a window instead of the full causal mask.
        _window("window_train_fp16_d64", 4, 16, 16, 4096, 4096, 64, 1024, 4, "fp16", True),
        # Odd sizes: 11 sequences of 1,500 tokens, three query heads to a key head, no sinks.
        _window("window_train_bf16_ragged", 11, 12, 4, 1500, 1500, 128, 500, 0, "bf16", True, layout="tokens"),
        # One long prompt: the costliest forward.
        _window("window_prompt_bf16", 1, 32, 8, 16384, 16384, 128, 4096, 4, "bf16", False, layout="tokens"),
        # One token for each of 32 sequences over a 16-bit cache filled to different lengths.
        _window("window_one_token_bf16", 32, 32, 8, 1, 8192, 128, 2048, 4, "bf16", False, lens=True),
        # The page bookkeeping of one decoding step: 256 requests, one token each.
        _tables("tables_one_token", 256, 8192, 1, 16),
        # ... and of a step that takes in prompts: 64 requests of about 1,024 new tokens.
        _tables("tables_prompts", 64, 4096, 2048, 16),
        # The keys and values of one decoding step into the cache.
        _write("cache4_write_one_token", 64, 8, 128, 16, "bf16"),
        # ... and those of a long prompt.
        _write("cache4_write_prompt", 16384, 8, 128, 16, "bf16"),
        # One short request: a single token over 2,000 cached ones.
        _attend("cache4_attend_one_request", 1, 2000, 16, 4, 64, 16, 0, 0, "fp16"),
        # A full serving batch: 64 requests of up to 16,384 cached tokens.
        _attend("cache4_attend_batch", 64, 16384, 32, 8, 128, 16, 0, 0, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng):
    hk = rng.choice([1, 2, 3, 4, 8])
    return hk * rng.choice([1, 1, 2, 3, 4, 8]), hk


def _pairs(n, s, window, sinks):
    """Visible (query, key) pairs of one head, the queries being the last n of s positions."""
    total = 0
    for i in (range(s - n, s) if n <= 64 else ()):
        total += min(i + 1, window) + min(sinks, max(0, i + 1 - window))
    if n > 64:
        def upto(m):  # positions 0 .. m - 1
            full = min(m, window)
            band = full * (full + 1) // 2 + (m - full) * window
            rest = m - full  # positions with keys before the window: 1, 2, ... of them
            few = min(rest, sinks)
            return band + few * (few + 1) // 2 + (rest - few) * sinks
        total = upto(s) - upto(s - n)
    return total


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "window", "window", "window", "tables", "write", "attend", "attend"])
    if op == "norm_rope":
        h, hk = _heads(rng)
        d, dtype = rng.choice([16, 32, 64, 64, 128, 128]), rng.choice(["fp16", "bf16", "bf16", "fp32"])
        n = _log_int(rng, 1, 16384)
        most = 4 * 4096 * 40 * 128 * 2 // (DTYPES[dtype].itemsize * d * (h + hk))  # tokens of the largest case
        z = _log_int(rng, 1, max(1, min(256, most // n)))
        return _norm_rope(None, z, h, hk, n, d, dtype, rng.random() < 0.6, rng.choice(["tokens", "heads"]),
                          rng.random() < 0.3)
    if op == "window":
        h, hk = _heads(rng)
        d, dtype = rng.choice([32, 64, 64, 128, 128]), rng.choice(["fp16", "bf16"])
        sinks = rng.choice([0, 1, 4, 4, 16, 64])
        if rng.random() < 0.35:  # a few tokens over a cache
            s = _log_int(rng, 16, 32768)
            z = _log_int(rng, 1, max(1, min(128, (1 << 21) // (s * hk))))
            return _window(None, z, h, hk, rng.choice([1, 1, 1, 2, 5]), s, d, _log_int(rng, 16, 2 * s), sinks, dtype,
                           False, True, rng.choice(["heads", "tokens"]))
        s = _log_int(rng, 16, 16384)
        n = s if rng.random() < 0.7 else _log_int(rng, 1, s)
        window = _log_int(rng, 1, max(2, s))
        train = rng.random() < 0.6
        z = _log_int(rng, 1, max(1, min(64, 32768 // n)))
        most = 32 * _pairs(16384, 16384, 4096, 4) * 128
        while z > 1 and z * h * _pairs(n, s, window, sinks) * d * (3.5 if train else 1.0) > most:
            z //= 2
        if h * _pairs(n, s, window, sinks) * d * (3.5 if train else 1.0) > most:
            h, hk, train = hk, hk, False
        return _window(None, z, h, hk, n, s, d, window, sinks, dtype, train, False, rng.choice(["heads", "tokens"]))
    if op == "tables":
        return _tables(None, _log_int(rng, 1, 1024), _log_int(rng, 1, 16384), _log_int(rng, 1, 64),
                       rng.choice([16, 32, 64, 128]))
    if op == "write":
        hk, d = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128])
        return _write(None, _log_int(rng, 1, 16384), hk, d, rng.choice([16, 32, 64, 128]), rng.choice(["fp16", "bf16"]))
    h, hk = _heads(rng)
    longest = _log_int(rng, 16, 32768)
    requests = _log_int(rng, 1, max(1, min(256, 64 * 16384 * 8 // (longest * hk))))
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 8192), rng.choice([0, 4]))])
    return _attend(None, requests, longest, h, hk, rng.choice([32, 64, 128]), rng.choice([16, 32, 64]), window, sinks,
                   rng.choice(["fp16", "bf16"]))


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _view(case, heads, length, dtype, g, outliers=False):
    """[z, heads, length, d] in the case's layout, drawn N(0, 1); every eighth channel eight times as large."""
    z, d = case["z"], case["d"]
    shape = (z, length, heads, d) if case["layout"] == "tokens" else (z, heads, length, d)
    t = torch.randn(shape, device="cuda", dtype=dtype, generator=g)
    if outliers:
        t[..., ::8] *= 8
    return t.transpose(1, 2) if case["layout"] == "tokens" else t


def _norm_rope_inputs(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    z, n, d = case["z"], case["n"], case["d"]
    q, k = (_view(case, case[x], n, dtype, g, True) for x in ("h", "hk"))
    qw, kw = ((1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dtype) for _ in range(2))
    dq, dk = (_view(case, case[x], n, dtype, g) for x in ("h", "hk"))
    rows = max(n, 16384)
    angles = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d // 2))
    start = torch.randint(0, rows - n + 1, (z, 1), device="cuda", generator=g)
    positions = (start + torch.arange(n, device="cuda")).to(torch.int32)
    return {"q": q, "k": k, "qw": qw, "kw": kw, "dq": dq, "dk": dk, "cos": angles.cos().float(),
            "sin": angles.sin().float(), "positions": positions}


def _window_inputs(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    q = _view(case, case["h"], case["n"], dtype, g)
    k, v = (_view(case, case["hk"], case["s"], dtype, g) for _ in range(2))
    do = _view(case, case["h"], case["n"], dtype, g)
    lens = None
    if case["lens"]:
        lens = torch.randint(max(1, case["s"] // 4), case["s"] + 1, (case["z"],), device="cuda", generator=g,
                             dtype=torch.int32).clamp_(min=min(case["n"], case["s"]))
    return {"q": q, "k": k, "v": v, "do": do, "lens": lens}


def _pages_of(lens, page, g, spare=0):
    """Table [requests, widest] of page numbers in random order (-1 where a request has none), their total, and
    `spare` more numbers."""
    need = (lens + page - 1) // page
    total = int(need.sum())
    order = torch.randperm(total + spare, device="cuda", generator=g).to(torch.int32)
    width = max(1, int(need.max()))
    at = torch.arange(width, device="cuda")[None]
    first = torch.cumsum(need, 0) - need
    table = torch.where(at < need[:, None], order[(first[:, None] + at).clamp(max=total + spare - 1)], -1)
    return table.to(torch.int32), total, order[total:]


def _tables_inputs(case, seed):
    g, r, page = _gen(seed), case["requests"], case["page"]
    lens = torch.randint(0, case["longest"] + 1, (r,), device="cuda", generator=g)
    tokens = r * (1 + case["new"]) // 2  # the step's size, shared out unevenly: at most 1.5 * new for a request
    share = 0.5 + torch.rand(r, device="cuda", dtype=torch.float64, generator=g)
    new = 1 + (share / share.sum() * (tokens - r)).floor().long()
    spare = int(((new + page - 1) // page + 1).sum())
    table, _, free = _pages_of(lens, page, g, spare)
    width = (case["longest"] + 2 * case["new"] + page - 1) // page
    wide = torch.full((r, width), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return {"lens": lens.to(torch.int32), "new": new.to(torch.int32), "tables": wide, "free": free.contiguous(),
            "tokens": tokens + 8}


def _write_inputs(case, seed):
    g, t = _gen(seed), case["tokens"]
    kv = torch.randn((t, 2, case["hk"], case["d"]), device="cuda", dtype=DTYPES[case["dtype"]], generator=g)
    kv[..., ::8] *= 4
    pages = (t + case["page"] - 1) // case["page"] + 1  # the last page stays free
    slots = torch.randperm(pages - 1, device="cuda", generator=g)[:, None] * case["page"]
    slots = (slots + torch.arange(case["page"], device="cuda")).reshape(-1)[:t].contiguous()
    slots[t - t // 16:] = -1  # a batch padded behind its last token
    return {"k": kv[:, 0], "v": kv[:, 1], "slots": slots, "pages": pages}


def _attend_inputs(case, seed):
    """The cache's bytes, made directly: random codes, exponents of values near 1."""
    g, r, page, hk, d = _gen(seed), case["requests"], case["page"], case["hk"], case["d"]
    low = max(1, case["longest"] // 4)
    lens = torch.randint(low, case["longest"] + 1, (r,), device="cuda", generator=g)
    table, pages, _ = _pages_of(lens, page, g)
    codes = torch.randint(0, 256, (pages, hk, 2, page, d // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.randint(124, 127, (pages, hk, 2, page, d // 32), device="cuda", generator=g, dtype=torch.uint8)
    q = torch.randn((r, case["h"], d), device="cuda", dtype=DTYPES[case["dtype"]], generator=g)
    return {"q": q, "codes": codes, "scales": scales, "tables": table, "lens": lens.to(torch.int32)}


_INPUTS = {"norm_rope": _norm_rope_inputs, "window": _window_inputs, "tables": _tables_inputs,
           "write": _write_inputs, "attend": _attend_inputs}


def prepare(case, seed):
    state = dict(_INPUTS[case["op"]](case, seed), case=case)
    op = case["op"]
    if op == "norm_rope" and case["train"]:
        for name in ("q", "k", "qw", "kw"):
            state[name].requires_grad_()
    if op == "window" and case["train"]:
        for name in ("q", "k", "v"):
            state[name].requires_grad_()
    if op == "write":
        if own:
            state["cache"] = _tattn().Cache4.empty(state["pages"], case["page"], case["hk"], case["d"],
                                                   dtype=DTYPES[case["dtype"]], device="cuda")
        else:
            state["values"] = torch.zeros((state["pages"] * case["page"], 2, case["hk"], case["d"]), device="cuda")
    if op == "attend" and own:
        state["cache"] = _tattn().Cache4(state["codes"], state["scales"], dtype=DTYPES[case["dtype"]])
    return state


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    tattn, op = _tattn(), case["op"]
    if op == "norm_rope":
        q, k = tattn.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["positions"], eps=EPS,
                                  interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"]))
        return dict(zip(("q", "k", "dq", "dk", "dqw", "dkw"), (q.detach(), k.detach(), *grads)))
    if op == "window":
        o = tattn.window_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"], lens=s["lens"])
        if not case["train"]:
            return {"o": o}
        grads = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))
    if op == "tables":
        slots, positions, starts, taken = tattn.page_tables(s["lens"], s["new"], s["tables"], s["free"], case["page"],
                                                            s["tokens"])
        return {"tables": s["tables"], "slots": slots, "positions": positions, "starts": starts, "taken": taken}
    if op == "write":
        tattn.cache4_write(s["cache"], s["k"], s["v"], s["slots"])
        k, v = tattn.cache4_read(s["cache"], s["slots"])
        return {"k": k, "v": v}
    return {"o": tattn.cache4_attention(s["q"], s["cache"], s["tables"], s["lens"], window=case["window"] or None,
                                        sinks=case["sinks"])}


def _rotate(a, cos, sin, interleaved):
    """[z, heads, n, d] turned by the angles of [z, n, d / 2]."""
    cos, sin = cos[:, None], sin[:, None]
    out = torch.empty_like(a)
    x, y = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, a.shape[-1] // 2),
                                                                       slice(a.shape[-1] // 2, None))
    out[..., x] = a[..., x] * cos - a[..., y] * sin
    out[..., y] = a[..., y] * cos + a[..., x] * sin
    return out


def _plain_norm_rope(case, s):
    cos, sin = (s[x][s["positions"].long()] for x in ("cos", "sin"))
    out = {}
    for x, w, g in (("q", "qw", "dq"), ("k", "kw", "dk")):
        a, wt = s[x].detach().float(), s[w].detach().float()
        r = (a.square().mean(-1, keepdim=True) + EPS).rsqrt()
        out[x] = _rotate(a * r * wt, cos, sin, case["interleaved"]).to(s[x].dtype)
        if case["train"]:
            t = _rotate(s[g].float(), cos, -sin, case["interleaved"])
            a = a * r
            out["d" + w] = (t * a).sum((0, 1, 2)).to(s[w].dtype)
            t = t * wt
            out["d" + x] = ((t - a * (t * a).mean(-1, keepdim=True)) * r).to(s[x].dtype)
    return out


def _hidden(q_pos, k_pos, window, sinks):
    """Truth values [.., n, keys]: the keys that a query at its position does not see."""
    i, j = q_pos[..., :, None], k_pos[None, :]
    return (j > i) | ((i - j >= window) & (j >= sinks))


def _plain_window(case, s):
    """Blocks of queries over the keys that any of them sees: the first ones, and the window's."""
    z, h, hk, n, length, d = (case[x] for x in ("z", "h", "hk", "n", "s", "d"))
    window, sinks, g = case["window"], case["sinks"], h // hk
    scale, dtype = d ** -0.5, s["q"].dtype
    k, v = s["k"].detach().float(), s["v"].detach().float()
    if s["lens"] is not None:
        q = s["q"].float().reshape(z, hk, g * n, d)
        pos = s["lens"].long()[:, None] - n + torch.arange(n, device="cuda")
        hide = _hidden(pos, torch.arange(length, device="cuda"), window, sinks)
        p = (torch.matmul(q, k.transpose(2, 3).contiguous()) * scale).reshape(z, hk, g, n, length)
        p = p.masked_fill(hide[:, None, None], -math.inf)
        p = (p - p.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
        return {"o": torch.matmul(p.reshape(z, hk, g * n, length), v).reshape(z, h, n, d).to(dtype)}
    q, train = s["q"].detach().float().reshape(z, hk, g, n, d), case["train"]
    out = torch.empty((z, hk, g, n, d), device="cuda")
    if train:
        do = s["do"].float().reshape(z, hk, g, n, d)
        dq, dk, dv = torch.empty_like(out), torch.zeros_like(k), torch.zeros_like(v)
    rows, off = 1024, length - n
    for a in range(0, n, rows):
        b = min(a + rows, n)
        low = max(0, off + a - window + 1)
        first = min(sinks, low)
        keys = torch.cat((torch.arange(first, device="cuda"), torch.arange(low, off + b, device="cuda")))
        kb, vb = k[:, :, keys], v[:, :, keys]
        qb = q[:, :, :, a:b].reshape(z, hk, g * (b - a), d)
        hide = _hidden(torch.arange(off + a, off + b, device="cuda"), keys, window, sinks).repeat(g, 1)
        p = (torch.matmul(qb, kb.transpose(2, 3).contiguous()) * scale).masked_fill_(hide, -math.inf)
        p = (p - p.amax(-1, keepdim=True)).exp_()
        p /= p.sum(-1, keepdim=True)
        o = torch.matmul(p, vb)
        out[:, :, :, a:b] = o.reshape(z, hk, g, b - a, d)
        if train:
            gb = do[:, :, :, a:b].reshape(z, hk, g * (b - a), d)
            ds = (torch.matmul(gb, vb.transpose(2, 3).contiguous()) - (gb * o).sum(-1, keepdim=True)) * p * scale
            dq[:, :, :, a:b] = torch.matmul(ds, kb).reshape(z, hk, g, b - a, d)
            dkb = torch.matmul(ds.transpose(2, 3).contiguous(), qb)
            dvb = torch.matmul(p.transpose(2, 3).contiguous(), gb)
            for total, part in ((dk, dkb), (dv, dvb)):
                total[:, :, :first] += part[:, :, :first]
                total[:, :, low:off + b] += part[:, :, first:]
    o = out.reshape(z, h, n, d).to(dtype)
    if not train:
        return {"o": o}
    return {"o": o, "dq": dq.reshape(z, h, n, d).to(dtype), "dk": dk.to(dtype), "dv": dv.to(dtype)}


def _plain_tables(case, s):
    page, tokens = case["page"], s["tokens"]
    lens, new, tables = s["lens"].long(), s["new"].long(), s["tables"]
    have = (lens + page - 1) // page
    need = (lens + new + page - 1) // page - have
    first = torch.cumsum(need, 0) - need
    at = torch.arange(tables.shape[1], device="cuda")[None] - have[:, None]
    fresh = (at >= 0) & (at < need[:, None])
    tables.copy_(torch.where(fresh, s["free"][(first[:, None] + at).clamp(0, s["free"].numel() - 1)], tables))
    ends = torch.cumsum(new, 0)
    t = torch.arange(tokens, device="cuda")
    r = torch.searchsorted(ends, t, right=True)
    real = r < lens.numel()
    r = r.clamp(max=lens.numel() - 1)
    pos = torch.where(real, lens[r] + t - (ends - new)[r], 0)
    slots = torch.where(real, tables[r, pos // page].long() * page + pos % page, -1)
    starts = torch.zeros(lens.numel() + 1, dtype=torch.int32, device="cuda")
    starts[1:] = ends
    return {"tables": tables, "slots": slots, "positions": pos.to(torch.int32), "starts": starts,
            "taken": need.sum().to(torch.int32).reshape(1)}


def _nearest_level(x):
    """Magnitudes up to 7 to the nearest level, ties to the one with an even mantissa."""
    low = torch.round(x * 2) * 0.5  # steps of a half up to 2, whole ones to 4, two from there
    mid = torch.round(x)
    high = torch.round(x * 0.5) * 2
    return torch.where(x < 2, low, torch.where(x < 4, mid, high)).clamp_(max=6)


def _power_of_two(biased):
    return (biased.to(torch.int32) << 23).view(torch.float32)


def _as_held(x):
    """[.., d] values as the cache holds them."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # amax = m 2^e, m in [0.5, 1)
    e = e - 3 + (m >= 0.875).to(e.dtype)
    scale = _power_of_two(e + 127)
    return (torch.copysign(_nearest_level(b.abs() / scale), b) * scale).reshape(x.shape)


def _plain_write(case, s):
    slots, values, dtype = s["slots"], s["values"], s["k"].dtype
    keep = slots >= 0
    at = torch.where(keep, slots, values.shape[0] - 1)  # on the free page
    held = _as_held(torch.stack((s["k"], s["v"]), 1).float())
    old = values[at]
    values[at] = torch.where(keep[:, None, None, None], held, old)
    got = torch.where(keep[:, None, None, None], values[at], 0.0).to(dtype)
    return {"k": got[:, 0].contiguous(), "v": got[:, 1].contiguous()}


def _plain_attend(case, s):
    """The requests' pages gathered, turned into values, and attended over in the table's order."""
    h, hk, d, page = case["h"], case["hk"], case["d"], case["page"]
    window, sinks = case["window"] or case["longest"], case["sinks"]
    level = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device="cuda")
    out = torch.empty(s["q"].shape, device="cuda", dtype=s["q"].dtype)
    some = max(1, (1 << 29) // (s["tables"].shape[1] * page * hk * d))  # requests at a time: 2 GiB of float32 keys
    for a in range(0, case["requests"], some):
        table = s["tables"][a:a + some].long().clamp(min=0)
        r, width = table.shape
        c = s["codes"][table].permute(0, 2, 3, 1, 4, 5)  # [r, hk, 2, pages, page, d / 2]
        e = _power_of_two(s["scales"][table].permute(0, 2, 3, 1, 4, 5))
        x = torch.stack((level[(c & 15).int()], level[(c >> 4).int()]), -1)
        x = x.reshape(r, hk, 2, width * page, d // 32, 32) * e.reshape(r, hk, 2, width * page, d // 32, 1)
        k, v = (t.reshape(r, hk, width * page, d) for t in x.unbind(2))
        q = s["q"][a:a + some].float().reshape(r, hk, h // hk, d)
        p = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
        hide = _hidden(s["lens"][a:a + some].long()[:, None] - 1, torch.arange(width * page, device="cuda"), window, sinks)
        p = p.masked_fill(hide[:, None], -math.inf)
        p = (p - p.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
        out[a:a + some] = torch.matmul(p, v).reshape(r, h, d).to(out.dtype)
    return {"o": out}


def _run_plain(case, state):
    return {"norm_rope": _plain_norm_rope, "window": _plain_window, "tables": _plain_tables, "write": _plain_write,
            "attend": _plain_attend}[case["op"]](case, state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "norm_rope":
        size = DTYPES[case["dtype"]].itemsize
        x = case["z"] * case["n"] * (case["h"] + case["hk"]) * case["d"]
        angles = case["z"] * case["n"] * (4 + 4 * case["d"])  # a position, its cosines and sines
        # x in, y out; training reads x again and dy, and writes dx.
        return {"bytes": float(x * size * (5 if case["train"] else 2) + angles), "flops": x * (30.0 if case["train"] else 10.0)}
    if op == "window":
        z, h, hk, n, s, d = (case[x] for x in ("z", "h", "hk", "n", "s", "d"))
        mean = s if not case["lens"] else (max(1, s // 4) + s) // 2
        pairs = _pairs(min(n, mean), mean, case["window"], case["sinks"])
        seen = min(mean, case["window"] + n - 1 + case["sinks"])
        io = 2.0 * d * z * (2 * h * n + 2 * hk * seen)
        # Training reads q, k, v, do and o once more, and writes three gradients.
        extra = 2.0 * d * z * (4 * h * n + 4 * hk * seen) if case["train"] else 0.0
        return {"bytes": io + extra, "flops": 4.0 * z * h * pairs * d * (3.5 if case["train"] else 1.0)}
    if op == "tables":
        r = case["requests"]
        tokens = r * (1 + case["new"]) / 2
        fresh = tokens / case["page"]
        return {"bytes": 12.0 * r + 8 * fresh + 16 * tokens, "flops": 8.0 * tokens}
    if op == "write":
        x = case["tokens"] * 2 * case["hk"] * case["d"]
        # Values in, codes out; codes in, values out.
        return {"bytes": x * (2 * 2 + 2 * 17 / 32) + 8.0 * case["tokens"], "flops": 6.0 * x}
    mean = (max(1, case["longest"] // 4) + case["longest"]) / 2
    seen = min(mean, case["window"] + case["sinks"]) if case["window"] else mean
    keys = case["requests"] * seen
    return {"bytes": keys * case["hk"] * case["d"] * 2 * 17 / 32 + 4.0 * case["requests"] * case["h"] * case["d"],
            "flops": 4.0 * keys * case["h"] * case["d"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _exact_norm_rope(case, seed):
    s = _norm_rope_inputs(case, seed)
    d, out = case["d"], {}
    angle = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]

    def turn(x, by):
        if case["interleaved"]:
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], d // 2, 2).contiguous()) * by).flatten(-2)
        c = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * by
        return torch.cat((c.real, c.imag), -1)

    for x, w, g in (("q", "qw", "dq"), ("k", "kw", "dk")):
        a, wt = s[x].double(), s[w].double()
        norm = torch.sqrt((a * a).sum(-1, keepdim=True) / d + EPS)
        out[x] = turn(a / norm * wt, angle)
        if case["train"]:
            t = turn(s[g].double(), angle.conj())
            out["d" + w] = (t * a / norm).sum((0, 1, 2))
            out["d" + x] = t * wt / norm - a * (t * wt * a).sum(-1, keepdim=True) / (d * norm ** 3)
    return {name: out[name] for name in (("q", "k", "dq", "dk", "dqw", "dkw") if case["train"] else ("q", "k"))}


def _exact_window(case, seed):
    """Slice by slice, from the materialised probabilities of 2,048 queries at a time."""
    s = _window_inputs(case, seed)
    z, h, hk, n, length, d = (case[x] for x in ("z", "h", "hk", "n", "s", "d"))
    if case["z"] * h * _pairs(n, length, case["window"], case["sinks"]) * d * (3.5 if case["train"] else 1) > 4e12:
        return None
    names = ("o", "dq", "dk", "dv") if case["train"] else ("o",)
    out = {x: torch.zeros((z, hk if x in ("dk", "dv") else h, length if x in ("dk", "dv") else n, d),
                          dtype=torch.float64, device="cuda") for x in names}
    scale = 1.0 / math.sqrt(d)
    ends = s["lens"].tolist() if s["lens"] is not None else [length] * z
    for b in range(z):
        end = ends[b]
        for top in range(0, n, 2048):
            rows = torch.arange(top, min(n, top + 2048), device="cuda")
            at = rows + (end - n)
            a0 = max(0, int(top + end - n) - case["window"] + 1)
            if a0 < case["sinks"]:
                a0 = 0
            cols = torch.cat((torch.arange(min(a0, case["sinks"]), device="cuda"),
                              torch.arange(a0, int(rows[-1]) + end - n + 1, device="cuda")))
            gap = at[:, None] - cols[None, :]
            seen = (gap >= 0) & ((gap < case["window"]) | (cols[None, :] < case["sinks"]))
            for head in range(h):
                kv = head * hk // h
                k, v = s["k"][b, kv, cols].double(), s["v"][b, kv, cols].double()
                q = s["q"][b, head, rows].double()
                w = torch.where(seen, torch.mm(q, k.t().contiguous()) * scale, -math.inf)
                w = torch.softmax(w, -1)
                o = torch.mm(w, v)
                out["o"][b, head, rows] = o
                if case["train"]:
                    t = s["do"][b, head, rows].double()
                    out["dv"][b, kv].index_add_(0, cols, torch.mm(w.t().contiguous(), t))
                    w = w * (torch.mm(t, v.t().contiguous()) - (t * o).sum(-1, keepdim=True)) * scale
                    out["dq"][b, head, rows] = torch.mm(w, k)
                    out["dk"][b, kv].index_add_(0, cols, torch.mm(w.t().contiguous(), q))
    return out


def _exact_write(case, seed):
    s = _write_inputs(case, seed)
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device="cuda")
    level = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    out = {}
    for name in ("k", "v"):
        x = s[name].double().reshape(case["tokens"], case["hk"], -1, 32)
        top = x.abs().amax(-1, keepdim=True)
        unit = torch.exp2(torch.floor(torch.log2(top)) - 2)
        unit = torch.where(top >= 8 * unit, 2 * unit, torch.where(top < 4 * unit, unit / 2, unit))  # log2's last bit
        unit = torch.where(top == 0, 1.0, torch.where(top >= 7 * unit, 2 * unit, unit))
        y = x.abs() / unit
        # The number of borders at or below y; on a border the level of even mantissa: below it for every other one.
        low, high = torch.bucketize(y, mid), torch.bucketize(y, mid, right=True)
        at = torch.where(low % 2 == 0, low, high)
        held = torch.where(x < 0, -level[at], level[at]) * unit
        held[s["slots"] < 0] = 0
        out[name] = held.reshape(case["tokens"], case["hk"], case["d"])
    return out


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    if case["requests"] * case["longest"] * case["hk"] * case["d"] > 1 << 31:
        return None
    h, hk, d = case["h"], case["hk"], case["d"]
    level = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    out = torch.empty((case["requests"], h, d), dtype=torch.float64, device="cuda")
    for r, end in enumerate(s["lens"].tolist()):
        j = torch.arange(end, device="cuda")
        if case["window"]:
            j = j[(j >= end - case["window"]) | (j < case["sinks"])]
        where, row = s["tables"][r, j // case["page"]].long(), j % case["page"]
        c = s["codes"][where, :, :, row].int()  # [keys, hk, 2, d / 2]
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
        x = torch.where(c < 8, 1.0, -1.0).double() * level[c & 7]
        unit = torch.exp2(s["scales"][where, :, :, row].double() - 127)
        x = (x.unflatten(-1, (-1, 32)) * unit[..., None]).flatten(-2)
        for kv in range(hk):
            q = s["q"][r, kv * (h // hk):(kv + 1) * (h // hk)].double()
            w = torch.softmax(torch.mm(q, x[:, kv, 0].t().contiguous()) / math.sqrt(d), -1)
            out[r, kv * (h // hk):(kv + 1) * (h // hk)] = torch.mm(w, x[:, kv, 1].contiguous())
    return {"o": out}


def _exact_tables(case, seed):
    """Counted on the host, request by request; whole numbers."""
    s, page = _tables_inputs(case, seed), case["page"]
    lens, new, free = (s[x].tolist() for x in ("lens", "new", "free"))
    tables = s["tables"].cpu()
    slots, positions, starts, used = [], [], [0], 0
    for r in range(len(lens)):
        for at in range(-(-lens[r] // page), -(-(lens[r] + new[r]) // page)):
            tables[r, at] = free[used]
            used += 1
        row = tables[r].tolist()
        for p in range(lens[r], lens[r] + new[r]):
            positions.append(p)
            slots.append(row[p // page] * page + p % page)
        starts.append(len(slots))
    pad = s["tokens"] - len(slots)
    out = {"tables": tables, "slots": torch.tensor(slots + [-1] * pad), "starts": torch.tensor(starts, dtype=torch.int32),
           "positions": torch.tensor(positions + [0] * pad, dtype=torch.int32),
           "taken": torch.tensor([used], dtype=torch.int32)}
    return {name: out[name].cuda() for name in ("tables", "slots", "positions", "starts", "taken")}


def exact(case, seed):
    return {"norm_rope": _exact_norm_rope, "window": _exact_window, "tables": _exact_tables, "write": _exact_write,
            "attend": _exact_attend}[case["op"]](case, seed)
