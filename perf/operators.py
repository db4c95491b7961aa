"""Serving operators as measurable cases: attention of one new token over a paged key-value cache,
the attention weight each cached key has received, eviction from the cache by that weight, and
penalties, biases and grammar masks on the logits.

``listed()`` names twelve cases, three or four for each operator; ``draw()`` makes more of the same
ranges.  Where ``own`` is true, ``run`` makes the calls a program makes of custom_flash_attn; where it
is false it computes the same in elementary torch operations.  Sizes are those of the GPT-2 family (12
to 25 heads of 64, contexts up to 1024, 50257 tokens) and generic ones: shared key-value heads, head
dims up to 128, caches up to 32768 rows, pages of 1 to 256 rows.

Case fields: ``op`` picks the operator, the others are its sizes and options.
"""
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
        # One token of one GPT-2 small sequence of a few hundred tokens, appended to its page: the
        # smallest step, launch and latency.
        dict(name="paged_single", op="paged", B=1, H=12, Hkv=12, D=64, N=400, page=16, dtype="bf16", sigma=1.0,
             rows_first=False, append=True, lse=False, weights=False),
        # One token of each of 32 GPT-2 XL sequences of very unequal lengths, one just begun among them.
        dict(name="paged_batch", op="paged", B=32, H=25, Hkv=25, D=64, N=1024, page=64, dtype="bf16", sigma=2.0,
             rows_first=False, append=True, lse=False, weights=False),
        # Long contexts, four query heads to a key-value head, head dim 128, fp16, with the log-sum-exp.
        dict(name="paged_long_shared", op="paged", B=4, H=32, Hkv=8, D=128, N=32768, page=128, dtype="fp16", sigma=1.0,
             rows_first=True, append=False, lse=True, weights=False),
        # A step that also adds each key's attention weight to its sum, as eviction by weight needs it.
        dict(name="paged_weights", op="paged", B=4, H=16, Hkv=16, D=64, N=4096, page=32, dtype="bf16", sigma=2.0,
             rows_first=False, append=True, lse=False, weights=True),
        # The weights of a short prompt's keys: GPT-2 small's heads.
        dict(name="weights_prompt", op="weights", B=1, H=12, Hkv=12, D=64, Nq=256, Nk=256, first=0, dtype="bf16",
             sigma=1.0, causal=True),
        # All queries of one long prompt: the largest piece of work here.
        dict(name="weights_long", op="weights", B=1, H=16, Hkv=16, D=64, Nq=8192, Nk=8192, first=0, dtype="bf16",
             sigma=2.0, causal=True),
        # Only the last queries of long prompts look back, shared heads, head dim 128, an odd length.
        dict(name="weights_window_shared", op="weights", B=2, H=32, Hkv=8, D=128, Nq=64, Nk=16001, first=15937,
             dtype="fp16", sigma=1.0, causal=True),
        # One GPT-2 small sequence cut to a small budget, ends inside pages.
        dict(name="evict_single", op="evict", B=1, Hkv=12, D=64, N=300, page=16, budget=130, recent=32, dtype="bf16",
             rows_first=False),
        # A batch of GPT-2 XL sequences at about their whole context, cut to half of it.
        dict(name="evict_batch", op="evict", B=16, Hkv=25, D=64, N=1024, page=64, budget=512, recent=128, dtype="bf16",
             rows_first=False),
        # Long prompts cut to an eighth, shared heads of 128, fp16.
        dict(name="evict_long", op="evict", B=4, Hkv=8, D=128, N=32768, page=128, budget=4096, recent=512, dtype="fp16",
             rows_first=True),
        # One sequence's logits, one penalty, short history.
        dict(name="logits_single", op="logits", B=1, V=50257, T=300, dtype="fp32", rows=False, bias="none", allowed=False),
        # A serving batch: each row its own penalties and history length, shared biases, grammar masks.
        dict(name="logits_batch", op="logits", B=128, V=50257, T=1024, dtype="fp32", rows=True, bias="shared", allowed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((12, 12), (16, 16), (20, 20), (25, 25), (32, 8), (32, 4), (28, 4), (24, 8), (16, 1))


def draw(rng):
    """One more case: caches of 1 to 32768 rows in pages of 1 to 256, batches of 1 to 64, every head
    layout; prompts of 16 to 8192 queries; budgets of a tenth to nine tenths of the cache; logits of
    1000 to 151936 tokens."""
    op = rng.choice(("paged", "paged", "paged", "weights", "weights", "evict", "evict", "logits", "logits"))
    c = dict(op=op)
    if op == "logits":
        c.update(B=_log_int(rng, 1, 128), V=_log_int(rng, 1000, 151936), T=_log_int(rng, 1, 8192),
                 dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), rows=rng.random() < 0.5,
                 bias=rng.choice(("none", "shared", "rows")), allowed=rng.random() < 0.5)
        while c["B"] * c["V"] > 128 * 50257:
            c["B"] = max(1, c["B"] // 2)
        return c
    H, Hkv = rng.choice(_HEADS)
    D = rng.choice((64, 64, 64, 128, 128, 32, 40, 80, 96))
    c.update(H=H, Hkv=Hkv, D=D, dtype=rng.choice(("bf16", "bf16", "fp16")))
    if op == "weights":
        c.update(B=rng.choice((1, 1, 2, 3)), sigma=rng.choice((1.0, 2.0)), causal=rng.random() < 0.8)
        n = _log_int(rng, 16, 8192)
        c.update(Nq=n, Nk=n, first=0)
        if rng.random() < 0.4:
            c["Nq"] = min(n, _log_int(rng, 1, 256))
            c["first"] = n - c["Nq"]
        while c["B"] * H * c["Nq"] * c["Nk"] * max(D, 64) > 16 * 8192 * 8192 * 64:
            c.update(Nq=max(1, c["Nq"] // 2), Nk=max(1, c["Nk"] // 2), first=c["first"] // 2)
        return c
    c.update(B=rng.choice((1, 1, 2, 4, 8, 16, 33, 64)), page=rng.choice((1, 8, 16, 16, 32, 48, 64, 64, 100, 128, 256)))
    n = _log_int(rng, 16, 32768)
    while c["B"] * Hkv * n * D > 4 * 8 * 32768 * 128:
        n //= 2
    c.update(N=max(2, n), rows_first=rng.random() < 0.4)
    if op == "paged":
        c.update(sigma=rng.choice((1.0, 2.0)), append=rng.random() < 0.7, lse=rng.random() < 0.4,
                 weights=rng.random() < 0.35)
    else:
        del c["H"]
        budget = max(1, int(c["N"] * rng.uniform(0.1, 0.9)))
        c.update(budget=budget, recent=int(budget * rng.choice((0.0, 0.1, 0.25, 0.5))))
    return c


# ---------------------------------------------------------------------------------------
# Inputs, from the seed alone.


def _randn(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * sigma).to(dtype)


def _lengths(case):
    """Cached rows per sequence: one as many as its table holds (less the row a step appends), the others
    spread from an eighth of that up, the last of a larger batch empty."""
    top = case["N"] - (1 if case.get("append") else 0)
    got = [top] + [max(1, int(top * (1 + 7 * (0.618034 * b % 1)) / 8)) for b in range(1, case["B"])]
    if case["B"] >= 8:
        got[-1] = 0
    return got


def _pool(rs, g, case, lengths, more, dtype, sigma):
    """Pages in random order with a few free ones, and each sequence's table (-1 where it has no page).
    The pool is (pages, heads, rows, dims): contiguous, or with `rows_first` views of the (pages, rows,
    heads, dims) buffers that programs keep which store a token's heads together."""
    page, cols = case["page"], -(-case["N"] // case["page"])
    need = [-(-n // page) for n in lengths]
    order = rs.permutation(sum(need) + more + 3)
    table = np.full((case["B"], cols), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (len(order), case["Hkv"], page, case["D"])
    if case["rows_first"]:
        shape = (shape[0], page, case["Hkv"], case["D"])
    k, v = _randn(g, shape, dtype, sigma), _randn(g, shape, dtype)
    if case["rows_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v, torch.from_numpy(table).to(DEV), order[at:]


def _sums(g, shape):
    """Attention sums as a cache has them: heavy-tailed, some keys never looked at, some equal."""
    w = torch.exp(2.0 * torch.randn(shape, generator=g, device=DEV) - 3.0)
    w = torch.where(w < 0.05, (w * 256).floor() / 256, w)
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.05, torch.zeros_like(w), w)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rs = np.random.Generator(np.random.PCG64(seed))
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    s = dict(case=case)
    if op == "paged":
        B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
        spare = 1 if case["append"] else 0
        lengths = _lengths(case)
        k, v, table, _ = _pool(rs, g, case, [n + spare for n in lengths], 0, dt, case["sigma"])
        s.update(k_pages=k, v_pages=v, table=table, lens=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                 q=_randn(g, (B, H, D), dt, case["sigma"]), k_new=None, v_new=None, sums=None)
        if spare:
            s.update(k_new=_randn(g, (B, Hkv, D), dt, case["sigma"]), v_new=_randn(g, (B, Hkv, D), dt))
        if case["weights"]:
            s["sums"] = _sums(g, (B, Hkv, table.shape[1] * case["page"]))
    elif op == "weights":
        B, H, Hkv, D, Nq, Nk = (case[n] for n in ("B", "H", "Hkv", "D", "Nq", "Nk"))
        # The (B, N, heads, D) projections, as views.
        q = _randn(g, (B, Nq, H, D), dt, case["sigma"]).transpose(1, 2)
        k = _randn(g, (B, Nk, Hkv, D), dt, case["sigma"]).transpose(1, 2)
        lse = torch.empty((B, H, Nq), dtype=torch.float32, device=DEV)
        for b in range(B):  # what the attention before it returned
            for h in range(H):
                x = (q[b, h].float() @ k[b, h // (H // Hkv)].float().T) / math.sqrt(D)
                if case["causal"]:
                    x.masked_fill_(_hidden(case), -INF)
                lse[b, h] = torch.logsumexp(x, -1)
        s.update(q=q, k=k, lse=lse)
    elif op == "evict":
        B, Hkv = case["B"], case["Hkv"]
        lengths = _lengths(case)
        cols = -(-case["budget"] // case["page"])
        k, v, table, free = _pool(rs, g, case, lengths, B * cols, dt, 1.0)
        new = torch.from_numpy(free[:B * cols].reshape(B, cols).astype(np.int32)).to(DEV)
        s.update(k_pages=k, v_pages=v, table=table, lens=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                 new_table=new, sums=_sums(g, (B, Hkv, table.shape[1] * case["page"])))
    else:
        B, V, T = case["B"], case["V"], case["T"]
        # A text repeats itself: token ids are far from uniform.
        u = torch.rand((B, T), generator=g, device=DEV)
        s.update(logits=_randn(g, (B, V), dt, 4.0), tokens=(V * u ** 4).long().clamp_(max=V - 1),
                 lengths=None, rep=1.2, pres=0.0, freq=0.0, bias=None, allowed=None)
        if case["rows"]:
            rand = lambda lo, hi: torch.rand(B, generator=g, device=DEV) * (hi - lo) + lo  # noqa: E731
            s.update(rep=rand(1.0, 1.5), pres=rand(0.0, 1.0), freq=rand(0.0, 0.5),
                     lengths=torch.from_numpy(rs.integers(0, T + 1, B).astype(np.int32)).to(DEV))
        if case["bias"] != "none":
            rows = B if case["bias"] == "rows" else 1
            b = _randn(g, (rows, V), torch.float32, 2.0)
            b = torch.where(torch.rand((rows, V), generator=g, device=DEV) < 0.9, torch.zeros_like(b), b)
            s["bias"] = b if case["bias"] == "rows" else b[0]
        if case["allowed"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g, device=DEV).to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------
# One pass.


def _fa():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tfg-flashattention_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import custom_flash_attn

    return custom_flash_attn


def _hidden(case):
    """The pairs of query and key that a causal mask hides: query i stands at position first + i."""
    at = torch.arange(case["Nq"], device=DEV)[:, None] + case["first"]
    return torch.arange(case["Nk"], device=DEV) > at


def _rows(pages, table):
    """(B, heads, rows, D) of each sequence's table, rows of absent pages being some others."""
    p = pages[table.clamp(min=0).long()]  # (B, columns, heads, page, D)
    B, C, H, R, D = p.shape
    return p.permute(0, 2, 1, 3, 4).reshape(B, H, C * R, D)


def _plain_paged(s):
    c = s["case"]
    k_pages, v_pages, table, lens = s["k_pages"], s["v_pages"], s["table"], s["lens"].long()
    B, H, Hkv, D, page = c["B"], c["H"], c["Hkv"], c["D"], c["page"]
    total = lens
    if c["append"]:
        at = table.long().gather(1, (lens // page)[:, None])[:, 0]
        k_pages[at, :, lens % page] = s["k_new"]
        v_pages[at, :, lens % page] = s["v_new"]
        total = lens + 1
    k, v = _rows(k_pages, table).float(), _rows(v_pages, table).float()
    q = s["q"].float().view(B, Hkv, H // Hkv, D)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    j = torch.arange(k.shape[2], device=DEV)
    x = torch.where((j < total[:, None])[:, None, None], x, -INF)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -INF, 0.0, m))
    z = p.sum(-1, keepdim=True)
    p = p / torch.where(z == 0, 1.0, z)
    out = {"o": (p @ v).view(B, H, D).to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = (m + torch.log(z)).view(B, H)
    if c["weights"]:
        w = p.sum(2)
        new = (j == lens[:, None])[:, None]
        s["sums"].copy_(torch.where(new, w, s["sums"] + w) if c["append"] else s["sums"] + w)
    return out


def _plain_weights(s):
    c = s["case"]
    G = c["H"] // c["Hkv"]
    q = s["q"].float().reshape(c["B"], c["Hkv"], G * c["Nq"], c["D"])
    x = (q @ s["k"].float().transpose(-1, -2)) * (1.0 / math.sqrt(c["D"]))
    x = x.view(c["B"], c["Hkv"], G, c["Nq"], c["Nk"])
    lse = s["lse"].view(c["B"], c["Hkv"], G, c["Nq"], 1)
    p = torch.exp(x - torch.where(lse == -INF, INF, lse))
    if c["causal"]:
        p = p.masked_fill(_hidden(c), 0.0)
    return p.sum((2, 3))


def _plain_evict(s):
    c = s["case"]
    k_pages, v_pages, table, new, page = s["k_pages"], s["v_pages"], s["table"].long(), s["new_table"].long(), c["page"]
    budget, lens, sums = c["budget"], s["lens"].long()[:, None, None], s["sums"]
    B, Hkv, N = sums.shape
    j = torch.arange(N, device=DEV)
    key = torch.where(j >= lens - c["recent"], INF, sums)
    key = torch.where(j < lens, key, -INF)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    i = torch.arange(budget, device=DEV)
    count = lens.clamp(max=budget)
    order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]), value=N)
    kept = torch.sort(torch.where(i < count, order, N), dim=-1).values
    live = kept < N
    kept = torch.where(live, kept, 0)
    at = table.clamp(min=0)[torch.arange(B, device=DEV)[:, None, None], kept // page]
    h = torch.arange(Hkv, device=DEV)[:, None]
    to = new[:, None, i // page].expand(B, Hkv, budget)
    for pages in (k_pages, v_pages):
        moved = torch.where(live[..., None], pages[at, h, kept % page], pages[to, h, i % page])
        pages[to, h, i % page] = moved
    weights = torch.where(live, sums.gather(2, kept), 0.0)
    return torch.where(live, kept, -1).int(), weights


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    tokens = s["tokens"]
    if s["lengths"] is not None:
        inside = torch.arange(tokens.shape[1], device=DEV) < s["lengths"][:, None]
        tokens = torch.where(inside, tokens, V)
    n = torch.zeros((B, V + 1), dtype=torch.int32, device=DEV)
    n = n.scatter_add_(1, tokens, torch.ones_like(tokens, dtype=torch.int32))[:, :V]
    rep, pres, freq = (p[:, None] if torch.is_tensor(p) else p for p in (s["rep"], s["pres"], s["freq"]))
    seen = n > 0
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * n - pres * seen
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEV)
        x = torch.where((s["allowed"][:, v // 32] >> (v % 32)) & 1 == 1, x, -INF)
    return x.to(s["logits"].dtype)


def run(s):
    c = s["case"]
    op = c["op"]
    if op == "paged":
        if own:
            got = _fa().decode_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["k_new"], s["v_new"],
                                     key_weights=s["sums"], return_lse=c["lse"])
            out = {"o": got[0], "lse": got[1]} if c["lse"] else {"o": got}
        else:
            out = _plain_paged(s)
        if c["weights"]:
            out["sums"] = s["sums"]
        if c["append"]:
            out.update(k_pages=s["k_pages"], v_pages=s["v_pages"])
        return out
    if op == "weights":
        if own:
            return _fa().key_weights(s["q"], s["k"], s["lse"], first_query=c["first"], causal=c["causal"])
        return _plain_weights(s)
    if op == "evict":
        if own:
            kept, weights = _fa().evict(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["sums"], s["new_table"],
                                        c["budget"], recent=c["recent"])
        else:
            kept, weights = _plain_evict(s)
        return {"kept": kept, "weights": weights, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if own:
        return _fa().penalize_logits(s["logits"], s["tokens"], lengths=s["lengths"], repetition=s["rep"],
                                     presence=s["pres"], frequency=s["freq"], bias=s["bias"], allowed=s["allowed"])
    return _plain_logits(s)


# ---------------------------------------------------------------------------------------
# What a pass cannot do without, and the definition in 64 bits.


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "logits":
        B, V = case["B"], case["V"]
        nbytes = 2 * B * V * size + 8 * B * case["T"]
        nbytes += {"none": 0, "shared": 4 * V, "rows": 4 * B * V}[case["bias"]] + (B * V / 8 if case["allowed"] else 0)
        return {"bytes": nbytes, "flops": 4 * B * V}
    D, Hkv, B = case["D"], case["Hkv"], case["B"]
    if op == "weights":
        H, Nq, Nk = case["H"], case["Nq"], case["Nk"]
        pairs = Nq * Nk
        if case["causal"]:
            pairs = sum(min(Nk, case["first"] + i + 1) for i in range(Nq))
        return {"bytes": size * B * D * (H * Nq + Hkv * Nk) + 4 * B * (H * Nq + Hkv * Nk), "flops": 2 * B * H * pairs * D}
    lengths = [n + (1 if case.get("append") else 0) for n in _lengths(case)]
    rows = sum(lengths) * Hkv
    if op == "paged":
        H = case["H"]
        nbytes = rows * 2 * D * size + 2 * B * H * D * size + (4 * B * Hkv * D * size if case["append"] else 0)
        return {"bytes": nbytes + (8 * rows if case["weights"] else 0), "flops": 4 * rows * (H // Hkv) * D}
    kept = sum(min(n, case["budget"]) for n in lengths) * Hkv
    return {"bytes": 4 * rows + kept * (4 * D * size + 8), "flops": 2 * rows}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "paged":
        return _exact_paged(s, case)
    if op == "weights":
        out = torch.zeros((case["B"], case["Hkv"], case["Nk"]), dtype=torch.float64, device=DEV)
        G, hide = case["H"] // case["Hkv"], _hidden(case) if case["causal"] else None
        for b in range(case["B"]):
            for h in range(case["H"]):
                x = torch.mm(s["q"][b, h].double(), s["k"][b, h // G].double().T.contiguous()) / case["D"] ** 0.5
                e = torch.exp(x - s["lse"][b, h].double()[:, None])
                out[b, h // G] += (e if hide is None else e * (~hide).double()).sum(0)
        return out
    if op == "evict":
        return _exact_evict(s, case)
    return _exact_logits(s, case)


def _exact_paged(s, case):
    page, G, D = case["page"], case["H"] // case["Hkv"], case["D"]
    k_pages, v_pages = s["k_pages"].clone(), s["v_pages"].clone()
    table, lens = s["table"].cpu().tolist(), s["lens"].cpu().tolist()
    o = torch.zeros((case["B"], case["H"], D), dtype=torch.float64, device=DEV)
    lse = torch.full((case["B"], case["H"]), -INF, dtype=torch.float64, device=DEV)
    sums = s["sums"].double() if case["weights"] else None
    for b, n in enumerate(lens):
        if case["append"]:
            k_pages[table[b][n // page], :, n % page] = s["k_new"][b]
            v_pages[table[b][n // page], :, n % page] = s["v_new"][b]
            if sums is not None:
                sums[b, :, n] = 0.0
            n += 1
        if n == 0:
            continue
        ids = table[b][:-(-n // page)]
        k = torch.cat([k_pages[i] for i in ids], 1)[:, :n].double()
        v = torch.cat([v_pages[i] for i in ids], 1)[:, :n].double()
        for h in range(case["Hkv"]):
            x = torch.mm(s["q"][b, h * G:(h + 1) * G].double(), k[h].T.contiguous()) / D ** 0.5
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, 1)
            w = torch.softmax(x, 1)
            o[b, h * G:(h + 1) * G] = torch.mm(w, v[h])
            if sums is not None:
                sums[b, h, :n] += w.sum(0)
    out = {"o": o}
    if case["lse"]:
        out["lse"] = lse
    if case["weights"]:
        out["sums"] = sums
    if case["append"]:
        out.update(k_pages=k_pages, v_pages=v_pages)
    return out


def _exact_evict(s, case):
    page, budget = case["page"], case["budget"]
    k_pages, v_pages = s["k_pages"].clone(), s["v_pages"].clone()
    lens, table, new = s["lens"].cpu().numpy(), s["table"].cpu().numpy(), s["new_table"].cpu().numpy()
    sums = s["sums"].double().cpu().numpy()
    kept = np.full((case["B"], case["Hkv"], budget), -1, np.int32)
    weights = np.zeros((case["B"], case["Hkv"], budget))
    for b, n in enumerate(lens):
        count, tail = min(n, budget), min(n, case["recent"])
        if count == 0:
            continue
        to = np.arange(count)
        for h in range(case["Hkv"]):
            old = n - tail
            best = np.lexsort((np.arange(old), -sums[b, h, :old]))[:count - tail]
            rows = np.sort(np.concatenate([best, np.arange(old, n)]))
            kept[b, h, :count], weights[b, h, :count] = rows, sums[b, h, rows]
            a, i = (torch.from_numpy(x.astype(np.int64)).to(DEV) for x in (table[b, rows // page], new[b, to // page]))
            r, t = (torch.from_numpy(x.astype(np.int64)).to(DEV) for x in (rows % page, to % page))
            for p in (k_pages, v_pages):
                p[i, h, t] = p[a, h, r]
    return {"kept": torch.from_numpy(kept).to(DEV), "weights": torch.from_numpy(weights), "k_pages": k_pages, "v_pages": v_pages}


def _exact_logits(s, case):
    B, V = case["B"], case["V"]
    x = s["logits"].double().cpu().numpy()
    tokens = s["tokens"].cpu().numpy()
    get = lambda p, b: float(p[b]) if torch.is_tensor(p) else p  # noqa: E731
    for b in range(B):
        t = tokens[b] if s["lengths"] is None else tokens[b, :int(s["lengths"][b])]
        n = np.bincount(t, minlength=V)
        hit = np.nonzero(n)[0]
        r = x[b, hit]
        r = np.where(r > 0, r / get(s["rep"], b), r * get(s["rep"], b))
        x[b, hit] = r - get(s["freq"], b) * n[hit] - get(s["pres"], b)
        if s["bias"] is not None:
            x[b] += (s["bias"] if s["bias"].dim() == 1 else s["bias"][b]).double().cpu().numpy()
        if s["allowed"] is not None:
            bits = np.unpackbits(s["allowed"][b].cpu().numpy().view(np.uint8), bitorder="little")[:V]
            x[b, bits == 0] = -INF
    return torch.from_numpy(x)
