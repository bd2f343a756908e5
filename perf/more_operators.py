"""Operators of models that attend to more than their own text, whose speed and results are measured as training
and serving programs call them:

  cross    `tattn.cross_attention`: queries over the states of an encoder, of another length, with or without the
           lengths of the encoder's padded sequences; grouped heads; training, whole passages, and one token
  prefix   `tattn.prefix_attention`: the newest tokens of sequences that share a long prefix, over that prefix and
           over the keys each of them has added
  rope     `tattn.qk_rope_axes`: rotation of queries and keys by positions on several axes (time, height, width),
           with the norms of the heads or without, and the gradients
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


@functools.lru_cache(maxsize=None)
def _tattn():
    pkg = str(Path(__file__).resolve().parent.parent / "triton-attn_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tattn

    return tattn


# ---- cases ---------------------------------------------------------------------------------------

def _cross(name, z, h, hk, n, s, d, dtype, train, lens, layout="heads"):
    return {"name": name, "op": "cross", "z": z, "h": h, "hk": hk, "n": n, "s": s, "d": d, "dtype": dtype,
            "train": train, "lens": lens, "layout": layout}


def _prefix(name, groups, members, h, hk, n, prefix, s, d, dtype, ragged=False):
    return {"name": name, "op": "prefix", "groups": groups, "members": members, "h": h, "hk": hk, "n": n,
            "prefix": prefix, "s": s, "d": d, "dtype": dtype, "ragged": ragged}


def _rope(name, z, h, hk, frames, height, width, d, axes, dtype, train, norm, interleaved=False, layout="tokens"):
    """frames x height x width tokens after one that starts the sequence; axes: pairs turned by each axis, as text."""
    return {"name": name, "op": "rope", "z": z, "h": h, "hk": hk, "frames": frames, "height": height, "width": width,
            "d": d, "axes": axes, "dtype": dtype, "train": train, "norm": norm, "interleaved": interleaved,
            "layout": layout}


def listed():
    return [
        # One decoding step of 32 sequences over encoder states of 375 to 1,500 positions.
        _cross("cross_one_token_bf16", 32, 32, 8, 1, 1500, 128, "bf16", False, True),
        # A training step of a decoder over padded encoder states, as the projections leave them.
        _cross("cross_train_fp16_padded", 8, 16, 16, 1024, 1500, 64, "fp16", True, True, "tokens"),
        # As many queries as states, grouped heads.
        _cross("cross_train_bf16_d128", 4, 32, 8, 4096, 4096, 128, "bf16", True, False),
        # Image tokens that read a short text: many queries, few keys, an odd number of them.
        _cross("cross_train_fp16_short_text", 16, 8, 8, 4096, 77, 64, "fp16", True, True, "tokens"),
        # A long passage over longer states: the costliest forward.
        _cross("cross_passage_bf16", 1, 32, 8, 8192, 16384, 128, "bf16", False, False),
        # A small model trained in float32.
        _cross("cross_train_fp32", 2, 8, 8, 500, 700, 64, "fp32", True, True),
        # Four answers to one short prompt: every launch is latency.
        _prefix("prefix_four_answers", 1, 4, 16, 4, 1, 1000, 64, 64, "fp16"),
        # 64 requests behind one long system prompt.
        _prefix("prefix_system_prompt_bf16", 1, 64, 32, 8, 1, 8192, 1024, 128, "bf16"),
        # 16 samples of each of 8 prompts of different lengths.
        _prefix("prefix_samples_bf16", 8, 16, 16, 4, 1, 4096, 2048, 128, "bf16", True),
        # One decoding step of 32 sequences.
        _rope("rope_one_token", 32, 16, 4, 0, 0, 0, 128, "16 24 24", "bf16", False, False),
        # A training step on short videos.
        _rope("rope_train_video_bf16", 2, 24, 24, 16, 30, 45, 128, "16 24 24", "bf16", True, False),
        # A training step on images, two axes, with the norms of the heads, neighbouring pairs.
        _rope("rope_train_image_norm_fp16", 16, 16, 16, 1, 64, 64, 64, "0 16 16", "fp16", True, True, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng):
    hk = rng.choice([1, 2, 3, 4, 8])
    return hk * rng.choice([1, 1, 2, 3, 4, 8]), hk


def draw(rng):
    op = rng.choice(["cross", "cross", "cross", "prefix", "prefix", "rope", "rope"])
    if op == "cross":
        h, hk = _heads(rng)
        d, dtype = rng.choice([16, 32, 64, 64, 128, 128]), rng.choice(["fp16", "bf16", "bf16", "fp32"])
        train = rng.random() < 0.6
        n = rng.choice([1, 1, _log_int(rng, 2, 64), *(_log_int(rng, 16, 8192),) * 4])
        s = _log_int(rng, 1, 16384)
        slow = 8 if dtype == "fp32" else 1  # what a float32 product costs
        most = 4 * 32 * 4096 * 4096 * 128 * 3.5
        cost = h * n * s * d * (3.5 if train else 1.0) * slow
        z = _log_int(rng, 1, max(1, min(64, int(most / cost), (1 << 29) // (hk * s * d * 4), (1 << 29) // (h * n * d * 4))))
        return _cross(None, z, h, hk, n, s, d, dtype, train, rng.random() < 0.6, rng.choice(["heads", "tokens"]))
    if op == "prefix":
        h, hk = _heads(rng)
        d, dtype = rng.choice([16, 32, 64, 64, 128, 128]), rng.choice(["fp16", "bf16"])
        groups, n = rng.choice([1, 1, 1, 2, 5, 8]), rng.choice([1, 1, 1, 2, 5])
        prefix, s = _log_int(rng, 1, 32768 // groups), _log_int(rng, 8, 4096)
        most = max(1, min(256, (1 << 19) // (s * hk), 64 * 32 * 32768 // (h * n * prefix * 8)) // groups)
        return _prefix(None, groups, _log_int(rng, 1, most), h, hk, n, prefix, s, d, dtype, rng.random() < 0.4)
    h, hk = _heads(rng)
    d, dtype = rng.choice([16, 32, 64, 64, 128, 128]), rng.choice(["fp16", "bf16", "bf16", "fp32"])
    pairs, count = d // 2, rng.choice([2, 3, 3, 4])
    cuts = sorted(rng.randint(0, pairs) for _ in range(count - 1)) + [pairs if rng.random() < 0.7 else pairs - pairs // 4]
    axes = " ".join(str(max(0, b - a)) for a, b in zip([0, *cuts], cuts))
    frames = rng.choice([0, 1, 1, rng.randint(2, 24)])
    height, width = _log_int(rng, 1, 64), _log_int(rng, 1, 90)
    n = 1 + frames * height * width
    most = 2 * 48 * 21601 * 128 * 2 // (DTYPES[dtype].itemsize * d * (h + hk))  # tokens of the largest case
    z = _log_int(rng, 1, max(1, min(256, most // n)))
    return _rope(None, z, h, hk, frames, height, width, d, axes, dtype, rng.random() < 0.6, rng.random() < 0.4,
                 rng.random() < 0.3, rng.choice(["tokens", "heads"]))


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _view(case, heads, length, dtype, g, z=None, outliers=False):
    """[z, heads, length, d] in the case's layout, drawn N(0, 1); every eighth channel eight times as large."""
    z, d, tokens = z or case["z"], case["d"], case.get("layout") == "tokens"
    t = torch.randn((z, length, heads, d) if tokens else (z, heads, length, d), device="cuda", dtype=dtype, generator=g)
    if outliers:
        t[..., ::8] *= 8
    return t.transpose(1, 2) if tokens else t


def _lengths(count, low, high, g):
    return torch.randint(low, high + 1, (count,), device="cuda", generator=g, dtype=torch.int32)


def _cross_inputs(case, seed):
    g, dtype, s = _gen(seed), DTYPES[case["dtype"]], case["s"]
    q = _view(case, case["h"], case["n"], dtype, g)
    k, v = (_view(case, case["hk"], s, dtype, g) for _ in range(2))
    do = _view(case, case["h"], case["n"], dtype, g)
    return {"q": q, "k": k, "v": v, "do": do, "lens": _lengths(case["z"], s // 4, s, g) if case["lens"] else None}


def _prefix_inputs(case, seed):
    g, dtype, groups = _gen(seed), DTYPES[case["dtype"]], case["groups"]
    z, p, s = groups * case["members"], case["prefix"], case["s"]
    q = _view(case, case["h"], case["n"], dtype, g, z)
    pk, pv = (_view(case, case["hk"], p, dtype, g, groups) for _ in range(2))
    k, v = (_view(case, case["hk"], s, dtype, g, z) for _ in range(2))
    lens = _lengths(z, max(1, s // 8), s, g).clamp_(min=min(case["n"], s))
    return {"q": q, "pk": pk, "pv": pv, "k": k, "v": v, "lens": lens,
            "prefix_lens": _lengths(groups, p // 2, p, g) if case["ragged"] else None}


def _pair_axes(case):
    """The axis of each pair, -1 where none turns it."""
    out = [a for a, count in enumerate(case["axes"].split()) for _ in range(int(count))]
    return tuple(out + [-1] * (case["d"] // 2 - len(out)))


def _rope_inputs(case, seed):
    g, dtype, d, z = _gen(seed), DTYPES[case["dtype"]], case["d"], case["z"]
    count, f, hh, w = len(case["axes"].split()), case["frames"], case["height"], case["width"]
    n = 1 + f * hh * w
    q, k = (_view(case, case[x], n, dtype, g, outliers=True) for x in ("h", "hk"))
    dq, dk = (_view(case, case[x], n, dtype, g) for x in ("h", "hk"))
    qw, kw = ((1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dtype) for _ in range(2))
    # The first token and the grid after it, from a start of the sequence's own: every axis goes on where the text
    # before it ended.
    at = torch.arange(f * hh * w, device="cuda")
    grid = torch.stack((at // max(1, hh * w), at // max(1, w) % max(1, hh), at % max(1, w), at % 7)) + 1
    grid = torch.cat((torch.zeros((4, 1), device="cuda", dtype=torch.int64), grid), 1)[:count]
    start = torch.randint(0, 8192, (1, z, 1), device="cuda", generator=g)
    positions = (start + grid[:, None]).to(torch.int32).contiguous()
    # Frequencies start anew in every axis.
    index = torch.tensor([sum(x == a for x in _pair_axes(case)[:i]) for i, a in enumerate(_pair_axes(case))], device="cuda",
                         dtype=torch.float64)
    size = torch.tensor([max(1, sum(x == a for x in _pair_axes(case))) for a in _pair_axes(case)], device="cuda",
                        dtype=torch.float64)
    rows = 8192 + 1 + max(f, hh, w, 8)
    angles = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-index / size)
    return {"q": q, "k": k, "dq": dq, "dk": dk, "qw": qw if case["norm"] else None, "kw": kw if case["norm"] else None,
            "cos": angles.cos().float(), "sin": angles.sin().float(), "positions": positions, "axes": _pair_axes(case)}


_INPUTS = {"cross": _cross_inputs, "prefix": _prefix_inputs, "rope": _rope_inputs}


def prepare(case, seed):
    state = dict(_INPUTS[case["op"]](case, seed), case=case)
    if case["op"] == "rope":
        state["columns"] = torch.tensor(state["axes"], device="cuda")
    if case.get("train"):
        for name in ("q", "k", "v", "qw", "kw"):
            if state.get(name) is not None:
                state[name].requires_grad_()
    return state


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    tattn, op = _tattn(), case["op"]
    if op == "cross":
        o = tattn.cross_attention(s["q"], s["k"], s["v"], lens=s["lens"])
        if not case["train"]:
            return {"o": o}
        grads = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))
    if op == "prefix":
        return {"o": tattn.prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lens"],
                                            prefix_lens=s["prefix_lens"])}
    q, k = tattn.qk_rope_axes(s["q"], s["k"], s["cos"], s["sin"], s["positions"], s["axes"],
                              interleaved=case["interleaved"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
    if not case["train"]:
        return {"q": q, "k": k}
    leaves = ("q", "k", "qw", "kw") if case["norm"] else ("q", "k")
    grads = torch.autograd.grad((q, k), [s[x] for x in leaves], (s["dq"], s["dk"]))
    return dict(zip(("q", "k", *("d" + x for x in leaves)), (q.detach(), k.detach(), *grads)))


def _softmax(p):
    """Over the last dimension; rows without a visible score give zeros."""
    top = p.amax(-1, keepdim=True)
    p = (p - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, 1.0, total))


def _plain_cross(case, s):
    """Blocks of queries over all keys."""
    z, h, hk, n, length, d = (case[x] for x in ("z", "h", "hk", "n", "s", "d"))
    g, scale, dtype, train = h // hk, d ** -0.5, s["q"].dtype, case["train"]
    q, k, v = s["q"].detach().float().reshape(z, hk, g, n, d), s["k"].detach().float(), s["v"].detach().float()
    hide = None
    if s["lens"] is not None:
        hide = (torch.arange(length, device="cuda") >= s["lens"][:, None])[:, None, None]
    kt = k.transpose(2, 3).contiguous()
    out = torch.empty((z, hk, g, n, d), device="cuda")
    if train:
        do, vt = s["do"].float().reshape(z, hk, g, n, d), v.transpose(2, 3).contiguous()
        dq, dk, dv = torch.empty_like(out), torch.zeros_like(k), torch.zeros_like(v)
    rows = max(1, min(n, (1 << 30) // (z * h * length)))
    for a in range(0, n, rows):
        b = min(n, a + rows)
        qb = q[:, :, :, a:b].reshape(z, hk, g * (b - a), d)
        p = torch.matmul(qb, kt) * scale
        if hide is not None:
            p = p.masked_fill_(hide, -math.inf)
        p = _softmax(p)
        o = torch.matmul(p, v)
        out[:, :, :, a:b] = o.reshape(z, hk, g, b - a, d)
        if train:
            gb = do[:, :, :, a:b].reshape(z, hk, g * (b - a), d)
            ds = (torch.matmul(gb, vt) - (gb * o).sum(-1, keepdim=True)) * p * scale
            dq[:, :, :, a:b] = torch.matmul(ds, k).reshape(z, hk, g, b - a, d)
            dk += torch.matmul(ds.transpose(2, 3).contiguous(), qb)
            dv += torch.matmul(p.transpose(2, 3).contiguous(), gb)
    o = out.reshape(z, h, n, d).to(dtype)
    if not train:
        return {"o": o}
    return {"o": o, "dq": dq.reshape(z, h, n, d).to(dtype), "dk": dk.to(dtype), "dv": dv.to(dtype)}


def _plain_prefix(case, s):
    """Scores over the prefix, a group's sequences in one product, beside those over each sequence's own keys."""
    groups, m, h, hk, n, length, own_keys, d = (case[x] for x in ("groups", "members", "h", "hk", "n", "prefix", "s", "d"))
    z, g, scale = groups * m, h // hk, d ** -0.5
    q = s["q"].float().reshape(groups, m, hk, g * n, d)
    pk, pv, k, v = (s[x].float() for x in ("pk", "pv", "k", "v"))
    grouped = q.transpose(1, 2).reshape(groups, hk, m * g * n, d)
    pos = s["lens"].long()[:, None] - n + torch.arange(n, device="cuda")  # [z, n]
    a = torch.matmul(grouped, pk.transpose(2, 3).contiguous()) * scale
    if s["prefix_lens"] is not None:
        a = a.masked_fill(torch.arange(length, device="cuda") >= s["prefix_lens"][:, None, None, None], -math.inf)
    a = a.reshape(groups, hk, m, g, n, length).transpose(1, 2).reshape(z, hk, g, n, length)
    a = a.masked_fill((pos < 0)[:, None, None, :, None], -math.inf)
    b = torch.matmul(q.reshape(z, hk, g * n, d), k.transpose(2, 3).contiguous()).reshape(z, hk, g, n, own_keys) * scale
    b = b.masked_fill((torch.arange(own_keys, device="cuda") > pos[..., None])[:, None, None], -math.inf)
    p = _softmax(torch.cat((a, b), -1))
    a = p[..., :length].reshape(groups, m, hk, g * n, length).transpose(1, 2).reshape(groups, hk, m * g * n, length)
    o = torch.matmul(a, pv).reshape(groups, hk, m, g * n, d).transpose(1, 2).reshape(z, hk, g * n, d)
    o = o + torch.matmul(p[..., length:].reshape(z, hk, g * n, own_keys), v)
    return {"o": o.reshape(z, h, n, d).to(s["q"].dtype)}


def _rotate(a, cos, sin, interleaved):
    """[z, heads, n, d] turned by the angles of [z, n, d / 2]."""
    cos, sin = cos[:, None], sin[:, None]
    out = torch.empty_like(a)
    x, y = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, a.shape[-1] // 2),
                                                                       slice(a.shape[-1] // 2, None))
    out[..., x] = a[..., x] * cos - a[..., y] * sin
    out[..., y] = a[..., y] * cos + a[..., x] * sin
    return out


def _plain_rope(case, s):
    columns = s["columns"]
    pos = s["positions"].long()[columns.clamp(min=0)].permute(1, 2, 0)  # [z, n, d / 2]
    pair = torch.arange(columns.numel(), device="cuda")
    cos = torch.where(columns < 0, 1.0, s["cos"][pos, pair])
    sin = torch.where(columns < 0, 0.0, s["sin"][pos, pair])
    out = {}
    for x, w, g in (("q", "qw", "dq"), ("k", "kw", "dk")):
        a, dtype = s[x].detach().float(), s[x].dtype
        if not case["norm"]:
            out[x] = _rotate(a, cos, sin, case["interleaved"]).to(dtype)
            if case["train"]:
                out["d" + x] = _rotate(s[g].float(), cos, -sin, case["interleaved"]).to(dtype)
            continue
        wt = s[w].detach().float()
        r = (a.square().mean(-1, keepdim=True) + EPS).rsqrt()
        out[x] = _rotate(a * r * wt, cos, sin, case["interleaved"]).to(dtype)
        if case["train"]:
            t = _rotate(s[g].float(), cos, -sin, case["interleaved"])
            a = a * r
            out["d" + w] = (t * a).sum((0, 1, 2)).to(s[w].dtype)
            t = t * wt
            out["d" + x] = ((t - a * (t * a).mean(-1, keepdim=True)) * r).to(dtype)
    return {x: out[x] for x in ("q", "k", "dq", "dk", "dqw", "dkw") if x in out}


def _run_plain(case, state):
    return {"cross": _plain_cross, "prefix": _plain_prefix, "rope": _plain_rope}[case["op"]](case, state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op, size = case["op"], DTYPES[case["dtype"]].itemsize
    d, h, hk = case["d"], case["h"], case["hk"]
    if op == "cross":
        z, n, s = case["z"], case["n"], case["s"]
        seen = (s // 4 + s) / 2 if case["lens"] else float(s)
        # q, k, v in, o out; training reads them and do again, and writes three gradients.
        rows, keys = z * h * n * d, z * hk * seen * d
        if not case["train"]:
            return {"bytes": size * (2 * rows + 2 * keys), "flops": 4.0 * z * h * n * seen * d}
        return {"bytes": size * (6 * rows + 4 * keys + 2 * z * hk * s * d), "flops": 14.0 * z * h * n * seen * d}
    if op == "prefix":
        groups, n, s = case["groups"], case["n"], case["s"]
        z = groups * case["members"]
        shared = case["prefix"] * (0.75 if case["ragged"] else 1.0)
        tail = (max(1, s // 8) + s) / 2
        return {"bytes": size * d * (2 * hk * (groups * shared + z * tail) + 2 * z * h * n),
                "flops": 4.0 * z * h * n * (shared + tail) * d}
    n = 1 + case["frames"] * case["height"] * case["width"]
    x = case["z"] * n * (h + hk) * d
    angles = case["z"] * n * (4 * len(case["axes"].split()) + 4 * d)  # positions, cosines and sines
    # x in, y out; training reads dy and writes dx, with norms it reads x again too.
    passes = 2 if not case["train"] else 5 if case["norm"] else 4
    return {"bytes": float(x * size * passes + angles), "flops": x * 3.0 * (1 + case["train"]) * (3 if case["norm"] else 1)}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _exact_cross(case, seed):
    """Head by head, from the materialised probabilities of 2,048 queries at a time."""
    z, h, hk, n, length, d = (case[x] for x in ("z", "h", "hk", "n", "s", "d"))
    if z * h * (n * length * d * (3.5 if case["train"] else 1) + 4e8) > 4e12:
        return None
    s = _cross_inputs(case, seed)
    names = ("o", "dq", "dk", "dv") if case["train"] else ("o",)
    out = {x: torch.zeros((z, hk if x in ("dk", "dv") else h, length if x in ("dk", "dv") else n, d),
                          dtype=torch.float64, device="cuda") for x in names}
    ends = s["lens"].tolist() if case["lens"] else [length] * z
    for b in range(z):
        end = min(ends[b], length)
        if end <= 0:
            continue
        for head in range(h):
            kv = head * hk // h
            k, v = s["k"][b, kv, :end].double(), s["v"][b, kv, :end].double()
            for top in range(0, n, 2048):
                rows = slice(top, min(n, top + 2048))
                q = s["q"][b, head, rows].double()
                w = torch.softmax(torch.mm(q, k.t().contiguous()) / math.sqrt(d), -1)
                o = torch.mm(w, v)
                out["o"][b, head, rows] = o
                if case["train"]:
                    t = s["do"][b, head, rows].double()
                    out["dv"][b, kv, :end] += torch.mm(w.t().contiguous(), t)
                    w = w * (torch.mm(t, v.t().contiguous()) - (t * o).sum(-1, keepdim=True)) / math.sqrt(d)
                    out["dq"][b, head, rows] = torch.mm(w, k)
                    out["dk"][b, kv, :end] += torch.mm(w.t().contiguous(), q)
    return out


def _exact_prefix(case, seed):
    """Sequence by sequence, the prefix laid before its own keys."""
    m, h, hk, n, d = (case[x] for x in ("members", "h", "hk", "n", "d"))
    z, g = case["groups"] * m, h // hk
    if z * hk * (case["prefix"] + case["s"]) * d * (g * n + 8) > 1 << 36:
        return None
    s = _prefix_inputs(case, seed)
    out = torch.zeros((z, h, n, d), dtype=torch.float64, device="cuda")
    shared = s["prefix_lens"].tolist() if case["ragged"] else [case["prefix"]] * case["groups"]
    for b, end in enumerate(s["lens"].tolist()):
        first = shared[b // m]
        k, v = (torch.cat((s["p" + x][b // m, :, :first], s[x][b, :, :end]), 1).double() for x in "kv")
        for i in range(n):
            seen = first + end - n + 1 + i
            if end - n + i < 0:
                continue
            q = s["q"][b, :, i].double().reshape(hk, g, d)
            w = torch.softmax(torch.matmul(q, k[:, :seen].transpose(1, 2).contiguous()) / math.sqrt(d), -1)
            out[b, :, i] = torch.matmul(w, v[:, :seen].contiguous()).reshape(h, d)
    return {"o": out}


def _exact_rope(case, seed):
    s, d = _rope_inputs(case, seed), case["d"]
    angle = torch.ones((case["z"], s["positions"].shape[2], d // 2), dtype=torch.complex128, device="cuda")
    for i, axis in enumerate(s["axes"]):
        if axis >= 0:
            at = s["positions"][axis].long()
            angle[..., i] = torch.complex(s["cos"][:, i].double()[at], s["sin"][:, i].double()[at])
    angle, out = angle[:, None], {}

    def turn(x, by):
        if case["interleaved"]:
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], d // 2, 2).contiguous()) * by).flatten(-2)
        c = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * by
        return torch.cat((c.real, c.imag), -1)

    for x in ("q", "k"):
        a = s[x].double()
        t = turn(s["d" + x].double(), angle.conj()) if case["train"] else None
        if not case["norm"]:
            out[x], out["d" + x] = turn(a, angle), t
            continue
        wt = s[x + "w"].double()
        norm = torch.sqrt((a * a).sum(-1, keepdim=True) / d + EPS)
        out[x] = turn(a / norm * wt, angle)
        if case["train"]:
            out["d" + x + "w"] = (t * a / norm).sum((0, 1, 2))
            out["d" + x] = t * wt / norm - a * (t * wt * a).sum(-1, keepdim=True) / (d * norm ** 3)
    return {x: out[x] for x in ("q", "k", "dq", "dk", "dqw", "dkw") if out.get(x) is not None}


def exact(case, seed):
    return {"cross": _exact_cross, "prefix": _exact_prefix, "rope": _exact_rope}[case["op"]](case, seed)
