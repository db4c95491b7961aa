"""Operators around a paged key-value cache as measurable cases: rotary positions (and their gradient), new
tokens' keys and values into pages, attention of several new tokens over the pages, and a decode step for
sequences that share a prefix.

``listed()`` names twelve cases, three for each operator; ``draw()`` makes more of the same ranges.  Where
``own`` is true, ``run`` makes the calls a program makes of custom_flash_attn; where it is false it computes the
same in elementary torch operations.  Sizes are those of the GPT-2 family (12 to 25 heads of 64, contexts up to
1024) and generic ones: shared key-value heads, head dims up to 128, caches up to 32768 rows, pages of 1 to 256.

Case fields: ``op`` picks the operator, the others are its sizes and options.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


def listed():
    return [
        # One token of each of 8 GPT-2 small sequences: the smallest call, launch and latency.
        dict(name="rotate_token", op="rotate", B=8, H=12, Hkv=12, D=64, N=1, rot=64, interleaved=False, scaling="none",
             factor=1.0, magnitude=1.0, first=700, dtype="bf16", grad=False),
        # A training step's queries and keys, GPT-2 XL's heads over whole contexts, and the gradients.
        dict(name="rotate_train", op="rotate", B=8, H=25, Hkv=25, D=64, N=1024, rot=64, interleaved=True, scaling="none",
             factor=1.0, magnitude=1.0, first=0, dtype="bf16", grad=True),
        # A long prompt of an odd length past the trained one: frequencies scaled by bands, half of each head rotated.
        dict(name="rotate_long", op="rotate", B=1, H=32, Hkv=8, D=128, N=32001, rot=64, interleaved=False, scaling="bands",
             factor=8.0, magnitude=1.2079, first=0, dtype="fp16", grad=False),
        # One token of each of 32 GPT-2 XL sequences of unequal lengths, rotated on the way with its queries.
        dict(name="append_token", op="append", B=32, H=25, Hkv=25, D=64, N=1, held=1000, page=64, rot=64, interleaved=False,
             queries=True, ragged=False, rows_first=False, dtype="bf16"),
        # A batch of prompts of unequal lengths into empty caches, no rotation (learned positions).
        dict(name="append_prompts", op="append", B=16, H=25, Hkv=25, D=64, N=1024, held=0, page=64, rot=0,
             interleaved=False, queries=False, ragged=True, rows_first=False, dtype="bf16"),
        # A long chunk of two prompts behind what is cached, shared heads of 128, with its queries.
        dict(name="append_chunk", op="append", B=2, H=32, Hkv=8, D=128, N=8192, held=8192, page=128, rot=128,
             interleaved=True, queries=True, ragged=False, rows_first=True, dtype="fp16"),
        # Four drafted tokens of each of 8 GPT-2 XL sequences, checked in one step.
        dict(name="attend_drafts", op="attend", B=8, H=25, Hkv=25, D=64, N=4, held=1020, page=64, causal=True, ragged=False,
             lse=False, rows_first=False, sigma=1.5, dtype="bf16"),
        # Prompts of unequal lengths, some behind a cached beginning: GPT-2 XL's heads.
        dict(name="attend_prompts", op="attend", B=8, H=25, Hkv=25, D=64, N=800, held=224, page=64, causal=True,
             ragged=True, lse=False, rows_first=False, sigma=2.0, dtype="bf16"),
        # One chunk of a long prompt, four query heads to a key-value head of 128: the largest piece of work here.
        dict(name="attend_chunk", op="attend", B=1, H=32, Hkv=8, D=128, N=2048, held=14336, page=128, causal=True,
             ragged=False, lse=True, rows_first=True, sigma=1.0, dtype="fp16"),
        # 8 samples of one GPT-2 small prompt: the smallest shared step.
        dict(name="shared_samples", op="shared", R=1, B=8, H=12, Hkv=12, D=64, prefix=900, N=100, page=16, append=True,
             lse=False, rows_first=False, sigma=1.0, dtype="bf16"),
        # 16 samples of each of 4 GPT-2 XL prompts.
        dict(name="shared_groups", op="shared", R=4, B=64, H=25, Hkv=25, D=64, prefix=700, N=324, page=64, append=True,
             lse=False, rows_first=False, sigma=2.0, dtype="bf16"),
        # 64 requests behind one long instruction text, shared heads of 128, with the log-sum-exp.
        dict(name="shared_long", op="shared", R=1, B=64, H=32, Hkv=8, D=128, prefix=32000, N=512, page=128, append=False,
             lse=True, rows_first=True, sigma=1.0, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((12, 12), (16, 16), (20, 20), (25, 25), (32, 8), (32, 4), (28, 4), (24, 8), (16, 1))


def draw(rng):
    """One more case: texts and caches of 1 to 32768 rows in pages of 1 to 256, batches of 1 to 64, every head
    layout, rotations of all or part of a head in both layouts, chunks of 1 to 8192 tokens, 2 to 64
    sequences behind a prefix."""
    op = rng.choice(("rotate", "append", "append", "attend", "attend", "attend", "shared", "shared", "shared"))
    H, Hkv = rng.choice(_HEADS)
    D = rng.choice((64, 64, 64, 128, 128, 32, 40, 80, 96))
    c = dict(op=op, H=H, Hkv=Hkv, D=D, dtype=rng.choice(("bf16", "bf16", "fp16")))
    if op in ("rotate", "append"):
        c.update(rot=rng.choice((D, D, D // 2, D // 4 * 2, 20)), interleaved=rng.random() < 0.5,
                 B=rng.choice((1, 2, 3, 8, 16, 33, 64)))
    if op == "rotate":
        c.update(N=_log_int(rng, 1, 32768), scaling=rng.choice(("none", "linear", "base", "bands")),
                 factor=rng.choice((1.5, 4.0, 16.0)), magnitude=rng.choice((1.0, 1.0, 1.1386)), first=_log_int(rng, 1, 1000000) - 1,
                 grad=rng.random() < 0.4)
        if rng.random() < 0.25:
            c["dtype"] = "fp32"
        while c["B"] * c["N"] * (H + Hkv) * D > 32000 * 40 * 128 // (2 if c["grad"] or c["dtype"] == "fp32" else 1):
            c["N"] = max(1, c["N"] // 2)
            c["B"] = max(1, c["B"] - 1)
        return c
    c.update(page=rng.choice((1, 8, 16, 16, 32, 48, 64, 64, 100, 128, 256)), rows_first=rng.random() < 0.4)
    if op == "append":
        c.update(N=rng.choice((1, _log_int(rng, 1, 8192))), held=_log_int(rng, 1, 16384) - 1, queries=rng.random() < 0.5,
                 ragged=rng.random() < 0.5)
        if rng.random() < 0.3:
            c.update(rot=0, queries=False)
        while c["B"] * (c["N"] + c["held"]) * Hkv * D > 2 * 16384 * 8 * 128:
            c.update(N=max(1, c["N"] // 2), held=c["held"] // 2)
        while c["queries"] and c["B"] * c["N"] * H * D > 2 * 8192 * 32 * 128:
            c["N"] = max(1, c["N"] // 2)
        return c
    c["sigma"] = rng.choice((1.0, 2.0))
    c["lse"] = rng.random() < 0.4
    if op == "attend":
        c.update(B=rng.choice((1, 1, 2, 3, 8, 17)), N=rng.choice((_log_int(rng, 1, 16), _log_int(rng, 16, 4096))),
                 held=_log_int(rng, 1, 32768) - 1, causal=rng.random() < 0.8, ragged=rng.random() < 0.4)
        if not c["causal"]:
            c["held"] = max(1, c["held"])
        while (c["B"] * H * c["N"] * (c["N"] + c["held"]) * max(D, 64) > 32 * 2048 * 16384 * 128
               or c["B"] * Hkv * (c["N"] + c["held"]) * D > 4 * 32768 * 8 * 128):
            c.update(N=max(1, c["N"] // 2), held=max(1, c["held"] // 2))
        return c
    R = rng.choice((1, 1, 1, 2, 4, 7))
    n = rng.choice((2, 3, 5, 8, 8, 16, 32, 64))
    c.update(R=R, B=R * n, prefix=_log_int(rng, 16, 32768), N=_log_int(rng, 2, 2048), append=rng.random() < 0.7)
    while (R * Hkv * c["prefix"] * D + c["B"] * Hkv * c["N"] * D > 40000 * 8 * 128
           or c["B"] * H * (c["prefix"] + c["N"]) * max(D, 64) > 64 * 32 * 32768 * 128):
        c.update(prefix=max(1, c["prefix"] // 2), N=max(2, c["N"] // 2))
    return c


# ---------------------------------------------------------------------------------------
# Inputs, from the seed alone.


def _randn(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * sigma).to(dtype)


def _frequencies(case):
    """Radians a position for each pair of dims, in 64 bits: 10000^(-2i / rot), scaled for longer contexts."""
    rot, factor = case["rot"], case.get("factor", 1.0)
    base, kind = 10000.0, case.get("scaling", "none")
    if kind == "base":
        base *= factor ** (rot / (rot - 2)) if rot > 2 else 1.0
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    if kind == "linear":
        f = f / factor
    if kind == "bands":  # of 8192 trained positions: whole from 32 turns on, divided by the factor up to one
        keep = ((8192 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f


def _spread(top, count, seed=0):
    """`count` lengths: one of `top`, the others spread from an eighth of it up."""
    return [top] + [max(min(top, 1), int(top * (1 + 7 * (0.618034 * (b + seed) % 1)) / 8)) for b in range(1, count)]


def _sizes(case):
    """Rows each sequence holds before the call, and its new tokens."""
    B = case["B"]
    if case["op"] == "shared":
        held = _spread(case["N"] - (1 if case["append"] else 0), B)
        if B >= 8:
            held[-1] = 0  # one just begun
        return held, [1 if case["append"] else 0] * B
    held = _spread(case["held"], B)
    if B >= 8:
        held[-1] = 0 if case.get("causal", True) else 1
    return held, (_spread(case["N"], B, 3) if case["ragged"] else [case["N"]] * B)


def _pool(rs, g, case, rows, cols, dtype, sigma):
    """Pages in random order with a few free ones, and tables (-1 where there is no page) of texts of `rows`, each at
    least one page.  The pool is (pages, heads, rows, dims): contiguous, or with `rows_first` views of the (pages,
    rows, heads, dims) buffers that programs keep which store a token's heads together."""
    page = case["page"]
    need = [[max(1, -(-n // page)) for n in group] for group in rows]
    order = rs.permutation(sum(map(sum, need)) + 3)
    tables, at = [], 0
    for group, c in zip(need, cols):
        table = np.full((len(group), c), -1, np.int32)
        for b, n in enumerate(group):
            table[b, :n] = order[at:at + n]
            at += n
        tables.append(torch.from_numpy(table).to(DEV))
    shape = (len(order), case["Hkv"], page, case["D"])
    if case["rows_first"]:
        shape = (shape[0], page, case["Hkv"], case["D"])
    k, v = _randn(g, shape, dtype, sigma), _randn(g, shape, dtype)
    if case["rows_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v, tables


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rs = np.random.Generator(np.random.PCG64(seed))
    dt, op = DTYPES[case["dtype"]], case["op"]
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    s = dict(case=case)
    # The projections of N tokens, (B, N, heads, D), as views.
    tokens = lambda n, h, sigma=1.0: _randn(g, (B, n, h, D), dt, sigma).transpose(1, 2)  # noqa: E731
    if op == "rotate":
        N = case["N"]
        s.update(f=_frequencies(case), q=tokens(N, H), k=tokens(N, Hkv))
        at = torch.arange(N, device=DEV) + case["first"]
        if N == 1:  # a step of texts of unequal lengths
            at = torch.from_numpy(rs.integers(0, case["first"] + 1, (B, 1))).to(DEV)
        s["positions"] = at.int()
        if case["grad"]:
            s.update(gq=tokens(N, H), gk=tokens(N, Hkv))
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    page = case["page"]
    held, new = _sizes(case)
    columns = lambda rows: max(1, -(-rows // page))  # noqa: E731
    rows = [[a + n for a, n in zip(held, new)]]
    cols = [columns(max(rows[0]))]
    sigma = case.get("sigma", 1.0)
    if op == "shared":
        prefix = _spread(case["prefix"], case["R"])
        rows, cols = [prefix] + rows, [columns(case["prefix"])] + cols
    k_pages, v_pages, tables = _pool(rs, g, case, rows, cols, dt, sigma)
    s.update(k_pages=k_pages, v_pages=v_pages, table=tables[-1], lens=_ints(held))
    if op == "shared":
        s.update(prefix_table=tables[0], prefix_lens=_ints(prefix), q=_randn(g, (B, H, D), dt, sigma), k_new=None, v_new=None)
        if case["append"]:
            s.update(k_new=_randn(g, (B, Hkv, D), dt, sigma), v_new=_randn(g, (B, Hkv, D), dt))
        return s
    N = case["N"]
    s["new"] = _ints(new) if case["ragged"] else None
    if op == "attend":
        s["q"] = tokens(N, H, sigma)
        return s
    s.update(k=tokens(N, Hkv), v=tokens(N, Hkv), q=tokens(N, H) if case["queries"] else None)
    if case["rot"]:
        s["f"] = _frequencies(case)
    return s


# ---------------------------------------------------------------------------------------
# One pass.


def _fa():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tfg-flashattention_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import custom_flash_attn

    return custom_flash_attn


@functools.lru_cache(maxsize=64)
def _rotary(rot, interleaved, scaling, factor, magnitude):
    """A model's rotation, which a program makes once."""
    more = {"none": {}, "linear": dict(scaling="linear", factor=factor), "base": dict(scaling="base", factor=factor),
            "bands": dict(scaling="bands", factor=factor, trained_length=8192, low=1.0, high=32.0)}[scaling]
    return _fa().Rotary(rot, 10000.0, interleaved=interleaved, magnitude=magnitude, device=DEV, **more)


def _rotary_of(c):
    return _rotary(c["rot"], c["interleaved"], c.get("scaling", "none"), c.get("factor", 1.0), c.get("magnitude", 1.0))


def _turned(x, positions, f, c):
    """x (B, heads, N, D) in 32 bits, rotated by positions (B or 1, N)."""
    rot, x = c["rot"], x.float()
    t = positions.double()[:, None, :, None] * f
    m = c.get("magnitude", 1.0)
    cos, sin = (torch.cos(t) * m).float(), (torch.sin(t) * m).float()
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_rotate(s):
    c = s["case"]
    at = s["positions"].view(-1, c["N"])
    return tuple(_turned(x, at, s["f"], c).to(x.dtype) for x in (s["q"], s["k"]))


def _plain_append(s):
    c = s["case"]
    k_pages, v_pages, table, page, N = s["k_pages"], s["v_pages"], s["table"].long(), c["page"], c["N"]
    lens = s["lens"].long()[:, None]
    at = lens + torch.arange(N, device=DEV)
    k, v, q = s["k"], s["v"], s["q"]
    if c["rot"]:
        k = _turned(k, at, s["f"], c).to(k.dtype)
        q = q if q is None else _turned(q, at, s["f"], c).to(q.dtype)
    i = torch.arange(N, device=DEV).expand(c["B"], N)
    if s["new"] is not None:  # rows past a text's last one stand for that one
        new = s["new"].long()[:, None]
        if q is not None:
            q = torch.where((i < new)[:, None, :, None], q, torch.zeros_like(q))
        i = torch.minimum(i, (new - 1).clamp(min=0))
    row = lens + i
    pid, off = table.gather(1, row // page), row % page
    for pool, x in ((k_pages, k), (v_pages, v)):
        x = x.transpose(1, 2).gather(1, i[..., None, None].expand(c["B"], N, c["Hkv"], c["D"]))
        pool[pid, :, off] = x
    out = {"k_pages": k_pages, "v_pages": v_pages}
    return out if q is None else {**out, "q": q}


def _rows(pages, table):
    """(B, heads, rows, D) of each text's table in 32 bits, rows of absent pages being some others."""
    p = pages[table.clamp(min=0).long()]  # (B, columns, heads, page, D)
    B, C, H, R, D = p.shape
    return p.permute(0, 2, 1, 3, 4).reshape(B, H, C * R, D).float()


def _plain_attend(s):
    c = s["case"]
    B, H, Hkv, D, N = c["B"], c["H"], c["Hkv"], c["D"], c["N"]
    G = H // Hkv
    k, v = _rows(s["k_pages"], s["table"]), _rows(s["v_pages"], s["table"])
    q = s["q"].float().reshape(B, Hkv, G * N, D)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    lens, i = s["lens"].long()[:, None], torch.arange(N, device=DEV)
    seen = lens + i + 1 if c["causal"] else lens.expand(B, N)
    seen = seen[:, None].expand(B, G, N).reshape(B, 1, G * N, 1)
    x = torch.where(torch.arange(k.shape[2], device=DEV) < seen, x, -INF)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -INF, 0.0, m))
    z = p.sum(-1, keepdim=True)
    o = ((p @ v) / torch.where(z == 0, 1.0, z)).view(B, H, N, D)
    lse = (m + torch.log(z)).view(B, H, N)
    if s["new"] is not None:
        there = i < s["new"][:, None, None]
        o, lse = torch.where(there[..., None], o, 0.0), torch.where(there, lse, -INF)
    o = o.to(s["q"].dtype)
    return {"o": o, "lse": lse} if c["lse"] else {"o": o}


def _plain_shared(s):
    c = s["case"]
    R, B, H, Hkv, D, page = c["R"], c["B"], c["H"], c["Hkv"], c["D"], c["page"]
    G, n = H // Hkv, B // R
    lens = s["lens"].long()
    if c["append"]:
        at = s["table"].long().gather(1, (lens // page)[:, None])[:, 0]
        s["k_pages"][at, :, lens % page] = s["k_new"]
        s["v_pages"][at, :, lens % page] = s["v_new"]
        lens = lens + 1
    kp, vp = _rows(s["k_pages"], s["prefix_table"]), _rows(s["v_pages"], s["prefix_table"])
    k, v = _rows(s["k_pages"], s["table"]), _rows(s["v_pages"], s["table"])
    scale = 1.0 / math.sqrt(D)
    q = s["q"].float().view(B, Hkv, G, D)
    together = q.view(R, n, Hkv, G, D).transpose(1, 2).reshape(R, Hkv, n * G, D)
    xp = (together @ kp.transpose(-1, -2)) * scale
    xp = torch.where((torch.arange(kp.shape[2], device=DEV) < s["prefix_lens"][:, None])[:, None, None], xp, -INF)
    xp = xp.view(R, Hkv, n, G, -1).transpose(1, 2).reshape(B, Hkv, G, -1)
    x = (q @ k.transpose(-1, -2)) * scale
    x = torch.where((torch.arange(k.shape[2], device=DEV) < lens[:, None])[:, None, None], x, -INF)
    m = torch.maximum(x.amax(-1, keepdim=True), xp.amax(-1, keepdim=True))
    at = torch.where(m == -INF, 0.0, m)
    p, pp = torch.exp(x - at), torch.exp(xp - at)
    z = p.sum(-1, keepdim=True) + pp.sum(-1, keepdim=True)
    pp = pp.view(R, n, Hkv, G, -1).transpose(1, 2).reshape(R, Hkv, n * G, -1)
    op = (pp @ vp).view(R, Hkv, n, G, D).transpose(1, 2).reshape(B, Hkv, G, D)
    o = ((p @ v + op) / torch.where(z == 0, 1.0, z)).view(B, H, D).to(s["q"].dtype)
    out = {"o": o}
    if c["lse"]:
        out["lse"] = (m + torch.log(z)).view(B, H)
    return out


def run(s):
    c = s["case"]
    op = c["op"]
    if op == "rotate":
        if own:
            q, k = _fa().rotate(s["q"], s["k"], s["positions"], _rotary_of(c))
        else:
            q, k = _plain_rotate(s)
        out = {"q": q.detach(), "k": k.detach()}
        if c["grad"]:
            out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return out
    if op == "append":
        if not own:
            return _plain_append(s)
        q = _fa().append_paged(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], lengths=s["new"],
                               rotary=_rotary_of(c) if c["rot"] else None, q=s["q"])
        out = {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        return out if s["q"] is None else {**out, "q": q}
    if op == "attend":
        if not own:
            return _plain_attend(s)
        got = _fa().attend_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], lengths=s["new"],
                                 causal=c["causal"], return_lse=c["lse"])
        return {"o": got[0], "lse": got[1]} if c["lse"] else {"o": got}
    if own:
        got = _fa().decode_shared(s["q"], s["k_pages"], s["v_pages"], s["prefix_table"], s["prefix_lens"], s["table"],
                                  s["lens"], s["k_new"], s["v_new"], return_lse=c["lse"])
        out = {"o": got[0], "lse": got[1]} if c["lse"] else {"o": got}
    else:
        out = _plain_shared(s)
    if c["append"]:
        out.update(k_pages=s["k_pages"], v_pages=s["v_pages"])
    return out


# ---------------------------------------------------------------------------------------
# What a pass cannot do without, and the definition in 64 bits.


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    if op == "rotate":
        n = B * case["N"] * (H + Hkv)
        passes = 2 if case["grad"] else 1
        return {"bytes": 2 * passes * n * D * size, "flops": 3 * passes * n * case["rot"]}
    held, new = _sizes(case)
    if op == "append":
        n, q = sum(new) * Hkv, sum(new) * H if case["queries"] else 0
        # (Of a caller's padded batch the output queries' rows are written whole.)
        wrote = B * case["N"] * H if case["queries"] else 0
        return {"bytes": size * D * (4 * n + q + wrote), "flops": 3 * case["rot"] * (n + q) + n}
    if op == "attend":
        pairs = sum(sum(h + i + 1 for i in range(n)) if case["causal"] else h * n for h, n in zip(held, new))
        rows = sum(h + n if case["causal"] else h for h, n in zip(held, new))
        nbytes = size * D * (2 * rows * Hkv + sum(new) * H + B * case["N"] * H) + (4 * B * case["N"] * H if case["lse"] else 0)
        return {"bytes": nbytes, "flops": 4 * pairs * H * D}
    prefix = _spread(case["prefix"], case["R"])
    rows = sum(h + n for h, n in zip(held, new))
    pairs = rows + sum(prefix) * (B // case["R"])
    nbytes = size * D * (2 * Hkv * (rows + sum(prefix)) + 2 * B * H + (2 * B * Hkv if case["append"] else 0))
    return {"bytes": nbytes + (4 * B * H if case["lse"] else 0), "flops": 4 * pairs * H * D}


def _exact_turned(x, positions, case, back=False):
    """x (heads, N, D) rotated pair by pair as complex numbers in 64 bits; back: by the angles' opposites."""
    rot = case["rot"]
    f = _frequencies(case)
    turn = torch.polar(torch.full((len(positions), rot // 2), float(case.get("magnitude", 1.0)), dtype=torch.float64, device=DEV),
                       torch.outer(positions.double(), -f if back else f))
    y = x.detach().double().clone()
    first = slice(0, rot, 2) if case["interleaved"] else slice(0, rot // 2)
    second = slice(1, rot, 2) if case["interleaved"] else slice(rot // 2, rot)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend, "shared": _exact_shared}[case["op"]](s, case)


def _exact_rotate(s, case):
    at = s["positions"].long().view(-1, case["N"])
    each = lambda x, back: torch.stack([_exact_turned(x[b], at[b % len(at)], case, back) for b in range(case["B"])])  # noqa: E731
    out = {"q": each(s["q"], False), "k": each(s["k"], False)}
    if case["grad"]:
        out.update(dq=each(s["gq"], True), dk=each(s["gk"], True))
    return out


def _exact_append(s, case):
    k_pages, v_pages, page = s["k_pages"].double(), s["v_pages"].double(), case["page"]
    table, (held, new) = s["table"].cpu().numpy(), _sizes(case)
    q = None if s["q"] is None else torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, (h, n) in enumerate(zip(held, new)):
        rows = np.arange(h, h + n)
        at = torch.from_numpy(rows).to(DEV)
        pid, off = torch.from_numpy(table[b, rows // page].astype(np.int64)).to(DEV), at % page
        k = _exact_turned(s["k"][b, :, :n], at, case) if case["rot"] else s["k"][b, :, :n].double()
        k_pages[pid, :, off] = k.transpose(0, 1)
        v_pages[pid, :, off] = s["v"][b, :, :n].double().transpose(0, 1)
        if q is not None:
            q[b, :, :n] = _exact_turned(s["q"][b, :, :n], at, case) if case["rot"] else s["q"][b, :, :n].double()
    out = {"k_pages": k_pages, "v_pages": v_pages}
    return out if q is None else {**out, "q": q}


def _text(pages, ids, rows):
    """(heads, rows, D) of a text whose pages are `ids`."""
    return torch.cat([pages[i] for i in ids], 1)[:, :rows].double() if rows else pages[0, :, :0].double()


def _exact_attend(s, case):
    B, H, N, D, page, G = case["B"], case["H"], case["N"], case["D"], case["page"], case["H"] // case["Hkv"]
    table, (held, new) = s["table"].tolist(), _sizes(case)
    o = torch.zeros((B, H, N, D), dtype=torch.float64, device=DEV)
    lse = torch.full((B, H, N), -INF, dtype=torch.float64, device=DEV)
    for b, (h, n) in enumerate(zip(held, new)):
        total = h + n if case["causal"] else h
        k, v = (_text(p, table[b][:-(-total // page)], total) for p in (s["k_pages"], s["v_pages"]))
        for head in range(H):
            x = torch.mm(s["q"][b, head, :n].double(), k[head // G].T.contiguous()) / D ** 0.5
            if case["causal"]:
                x.masked_fill_(torch.ones_like(x, dtype=torch.bool).triu_(h + 1), -INF)
            lse[b, head, :n] = torch.logsumexp(x, 1)
            o[b, head, :n] = torch.mm(torch.softmax(x, 1), v[head // G])
    return {"o": o, "lse": lse} if case["lse"] else {"o": o}


def _exact_shared(s, case):
    B, H, D, page, G = case["B"], case["H"], case["D"], case["page"], case["H"] // case["Hkv"]
    k_pages, v_pages = s["k_pages"].clone(), s["v_pages"].clone()
    table, shared, (held, _) = s["table"].tolist(), s["prefix_table"].tolist(), _sizes(case)
    prefix = _spread(case["prefix"], case["R"])
    o = torch.zeros((B, H, D), dtype=torch.float64, device=DEV)
    lse = torch.full((B, H), -INF, dtype=torch.float64, device=DEV)
    each = B // case["R"]
    before = [[_text(p, t[:-(-n // page)], n) for p in (k_pages, v_pages)] for t, n in zip(shared, prefix)]
    for b, n in enumerate(held):
        if case["append"]:
            k_pages[table[b][n // page], :, n % page] = s["k_new"][b]
            v_pages[table[b][n // page], :, n % page] = s["v_new"][b]
            n += 1
        k, v = (torch.cat((old, _text(p, table[b][:-(-n // page)], n)), 1)
                for old, p in zip(before[b // each], (k_pages, v_pages)))
        for kv in range(case["Hkv"]):
            heads = slice(kv * G, (kv + 1) * G)
            x = torch.mm(s["q"][b, heads].double(), k[kv].T.contiguous()) / D ** 0.5
            lse[b, heads] = torch.logsumexp(x, 1)
            o[b, heads] = torch.mm(torch.softmax(x, 1), v[kv])
    out = {"o": o}
    if case["lse"]:
        out["lse"] = lse
    if case["append"]:
        out.update(k_pages=k_pages, v_pages=v_pages)
    return out
