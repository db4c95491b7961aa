"""The serving operators (custom_flash_attn.decode_paged, key_weights, evict, penalize_logits) against
plain implementations in 64 bits on the same inputs (needs a GPU).

Tolerances count roundings, u = 2^-24 for float32 and half = torch.finfo(type).eps / 2 for one rounding to
the output's type, and are worst cases of the sums as they are written here:
  * a score is a float32 sum of D exact products, scaled: off by at most ex = (D + 4) u X, X the largest
    scale * sum |q_d k_d| of the row; taking it to the exponent in the log2 domain adds 4 u (|x| + |lse|);
  * a softmax weight is off by twice that relative to itself (e^(2e) - 1 <= 2.1 (2e) for e < 0.04, with the
    offset's own error cancelling against the sum's), sums of n terms by n u of their magnitudes.
"""
import math
import sys

import numpy as np
import pytest
import torch

import custom_flash_attn as fa
from custom_flash_attn import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _randn(shape, g, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g) * sigma).to(dtype).to(DEV)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


class Paged:
    """A pool whose pages are dealt to sequences in random order; everything no sequence may see is NaN."""

    def __init__(self, g, lens, H_kv, D, page, dtype, cols=None, spare=0, rows_first=False, sigma=1.5, extra=3):
        self.lens, self.page, self.D, self.H_kv, self.dtype = lens, page, D, H_kv, dtype
        need = [-(-(max(n, 0) + spare) // page) for n in lens]
        self.P = sum(need) + extra
        cols = cols or max(max(need), 1)
        order = torch.randperm(self.P, generator=g).tolist()
        shape = (self.P, page, H_kv, D) if rows_first else (self.P, H_kv, page, D)
        self.k = torch.full(shape, NAN, dtype=dtype, device=DEV)
        self.v = torch.full(shape, NAN, dtype=dtype, device=DEV)
        if rows_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        table = torch.full((len(lens), cols), 2 ** 31 - 9, dtype=torch.int32)
        self.rows = []
        at = 0
        for b, n in enumerate(lens):
            n = max(n, 0)
            table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
            at += need[b]
            k, v = _randn((H_kv, n, D), g, dtype, sigma), _randn((H_kv, n, D), g, dtype)
            self.rows.append((k, v))
            for j in range(0, n, page):
                pid, m = int(table[b, j // page]), min(page, n - j)
                self.k[pid, :, :m] = k[:, j:j + m]
                self.v[pid, :, :m] = v[:, j:j + m]
        self.free = order[at:]
        self.table = table.to(DEV)
        self.seqlens = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def row(self, pool, b, j):
        return pool[int(self.table[b, j // self.page]), :, j % self.page]


def attend(q, k, v, scale):
    """One query (H, D) over (H_kv, L, D): o, lse, weights summed over the group (H_kv, L) in 64 bits, and the
    error bounds of lse, of o (before its rounding) and of the weights."""
    H, D = q.shape
    H_kv, L, _ = k.shape
    G = H // H_kv
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    o, lse = torch.zeros(H, D, dtype=torch.float64), torch.full((H,), -INF, dtype=torch.float64)
    w = torch.zeros(H_kv, L, dtype=torch.float64)
    eo, el, ew = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(w)
    for h in range(H if L else 0):
        kk, vv = k[h // G], v[h // G]
        x = scale * (kk @ q[h])
        lse[h] = torch.logsumexp(x, 0)
        p = torch.softmax(x, 0)
        o[h] = p @ vv
        w[h // G] += p
        X = float((scale * (kk.abs() @ q[h].abs())).max())
        ex = (D + 4) * U * X + 4 * U * (float(x.abs().max()) + abs(float(lse[h])))
        el[h] = ex + (L + 16) * U + 2 * U * abs(float(lse[h]))
        eo[h] = (4.2 * ex + (L + 16) * U) * (p @ vv.abs())
        ew[h // G] += (4.2 * ex + (L + 16) * U) * p
    return o, lse, w, eo, el, ew


def _near(got, want, bound, what):
    d = (got.double().cpu() - want).abs()
    worst = float((d - bound).max()) if d.numel() else 0.0
    _say(f"  {what}: max off {float(d.max()) if d.numel() else 0:.3e}, at most {float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0:.2f} of its bound")
    assert torch.isfinite(got.double()).all() and worst <= 0, what


LENS = [0, 1, 15, 16, 17, 127, 128, 129, 700, 2500]


@pytest.mark.parametrize("H,H_kv,D,page,dtype,append,rows_first", [
    (12, 12, 64, 16, BF, True, False),
    (12, 12, 64, 64, HF, False, True),
    (8, 2, 128, 128, HF, True, True),
    (8, 2, 128, 48, BF, False, False),
    (25, 25, 64, 100, BF, True, False),
    (16, 1, 64, 1, BF, True, False),
    (24, 1, 96, 16, HF, True, False),     # two tiles of query heads
    (34, 2, 80, 7, BF, True, True),
    (3, 3, 8, 16, HF, True, False),
    (6, 2, 40, 256, BF, True, False),
    (4, 4, 72, 8, HF, False, False),
    (5, 5, 128, 33, BF, True, False),
])
def test_decode_paged_matches_64_bits(H, H_kv, D, page, dtype, append, rows_first):
    _say(f"paged H={H} H_kv={H_kv} D={D} page={page} {dtype} append={append}")
    g = _gen(H * 1000 + D + page)
    c = Paged(g, LENS, H_kv, D, page, dtype, spare=1 if append else 0, rows_first=rows_first)
    B = len(LENS)
    q = _randn((B, H, D), g, dtype, 1.5)
    kn, vn = (_randn((B, H_kv, D), g, dtype), _randn((B, H_kv, D), g, dtype)) if append else (None, None)
    k0, v0 = c.k.clone(), c.v.clone()
    o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, return_lse=True)
    torch.cuda.synchronize()
    assert o.dtype == dtype and o.shape == (B, H, D) and lse.shape == (B, H)
    for b, n in enumerate(LENS):
        k, v = c.rows[b]
        if append:
            k, v = torch.cat([k, kn[b][:, None]], 1), torch.cat([v, vn[b][:, None]], 1)
            c.row(k0, b, n).copy_(kn[b])
            c.row(v0, b, n).copy_(vn[b])
        ro, rl, _, eo, el, _ = attend(q[b], k, v, D ** -0.5)
        if k.shape[1] == 0:
            assert (o[b] == 0).all() and (lse[b] == -INF).all()
            continue
        _near(o[b], ro, eo + _half(dtype) * (ro.abs() + eo), f"L={n} o")
        _near(lse[b], rl, el, f"L={n} lse")
    as_bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(as_bits(c.k), as_bits(k0)) and torch.equal(as_bits(c.v), as_bits(v0)), "pool"


def test_decode_paged_takes_strides_out_and_scale():
    g = _gen(3)
    lens, H, H_kv, D = [70, 300], 8, 4, 64
    c = Paged(g, lens, H_kv, D, 32, BF, spare=1, cols=20)
    wide = _randn((2, H, D + 24), g, BF)
    q = wide[..., 8:D + 8]
    kv = _randn((2, 3, H_kv, D), g, BF)
    out = torch.zeros(H, 2, D + 8, dtype=BF, device=DEV)
    table = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)[:, :20]
    table.copy_(c.table)
    got = fa.decode_paged(q, c.k, c.v, table, c.seqlens, kv[:, 0], kv[:, 2], out=out.transpose(0, 1)[..., :D],
                          softmax_scale=0.3)
    assert got.data_ptr() == out.data_ptr()
    for b in range(2):
        k, v = (torch.cat([t, n[b][:, None]], 1) for t, n in zip(c.rows[b], (kv[:, 0], kv[:, 2])))
        ro, _, _, eo, _, _ = attend(q[b], k, v, 0.3)
        _near(out[:, b, :D], ro, eo + _half(BF) * (ro.abs() + eo), f"b={b}")
    assert (out[..., D:] == 0).all()


def test_decode_paged_equals_decode_of_a_contiguous_cache():
    """A contiguous cache is a pool with one page a sequence."""
    g = _gen(4)
    B, H, N, D = 3, 12, 800, 64
    q, k, v = _randn((B, H, D), g, BF), _randn((B, H, N, D), g, BF), _randn((B, H, N, D), g, BF)
    sl = torch.tensor([800, 1, 333], dtype=torch.int32, device=DEV)
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
    o, lse = fa.decode_paged(q, k, v, table, sl, return_lse=True)
    o2, lse2 = fa.decode(q, k, v, sl, return_lse=True)
    # decode rounds its softmax weights to bf16 for the product, and each output once.
    assert (o.double() - o2.double()).abs().max() <= 3 * _half(BF) * v.abs().max().double()
    assert (lse - lse2).abs().max() <= 1e-4


def test_decode_paged_marks_bad_lengths_and_pages():
    g = _gen(5)
    lens, H_kv, D, page = [200, 100, 90, 40, 64], 2, 64, 16
    for aligned in (16, 20):
        c = Paged(g, lens, H_kv, D, aligned, BF, spare=1, cols=14)
        table = c.table.clone()
        table[1, 3] = c.P          # one of its pages is past the pool
        table[2, 90 // aligned] = -1   # the page of its new row is missing
        sl = c.seqlens.clone()
        sl[3] = -5
        sl[4] = 14 * aligned       # full: no room for the new row
        q, kn, vn = (_randn((5, n, D), g, BF) for n in (4, H_kv, H_kv))
        k0, v0 = c.k.clone(), c.v.clone()
        sums = torch.full((5, H_kv, 14 * aligned), 7.0, device=DEV)
        o, lse = fa.decode_paged(q, c.k, c.v, table, sl, kn, vn, return_lse=True, key_weights=sums)
        torch.cuda.synchronize()
        _say(f"page {aligned}: nan rows {torch.isnan(lse).all(1).tolist()}")
        assert torch.isnan(o[1:]).all() and torch.isnan(lse[1:]).all()
        k, v = (torch.cat([t, n[0][:, None]], 1) for t, n in zip(c.rows[0], (kn, vn)))
        ro, rl, w, eo, el, ew = attend(q[0], k, v, D ** -0.5)
        _near(o[0], ro, eo + _half(BF) * (ro.abs() + eo), "good row")
        c.row(k0, 0, 200).copy_(kn[0])
        c.row(v0, 0, 200).copy_(vn[0])
        c.row(k0, 1, 100).copy_(kn[1])   # its own page is good
        c.row(v0, 1, 100).copy_(vn[1])
        assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))
        assert torch.equal(c.v.view(torch.int16), v0.view(torch.int16))
        # Sums of marked rows stay, but for the new row that was written (nothing was added to it).
        assert (sums[2:] == 7).all() and (sums[1, :, :100] == 7).all() and (sums[1, :, 100] == 0).all()
        assert (sums[1, :, 101:] == 7).all() and (sums[0, :, 201:] == 7).all()


@pytest.mark.parametrize("page", [16, 5])
def test_decode_paged_rows_without_a_finite_score(page):
    """Scores of -inf have weight 0; nothing but such scores gives O = 0 and LSE = -inf; scores of the type's
    lowest value are finite and share the weight."""
    g = _gen(6)
    D, L = 64, 150
    c = Paged(g, [L, L, L], 1, D, page, BF)
    k = [t.clone() for t, _ in c.rows]
    k[0][:] = -INF
    k[1][:, :149] = -INF
    k[1][:, 149] = 1.0
    k[2][:] = torch.finfo(BF).min / 64
    for b in range(3):
        for j in range(L):
            c.row(c.k, b, j).copy_(k[b][:, j])
    q = torch.ones(3, 2, D, dtype=BF, device=DEV)
    sums = torch.zeros(3, 1, c.table.shape[1] * page, device=DEV)
    o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, return_lse=True, key_weights=sums, softmax_scale=1.0)
    torch.cuda.synchronize()
    assert (o[0] == 0).all() and (lse[0] == -INF).all() and (sums[0] == 0).all()
    assert torch.equal(o[1, 0], c.rows[1][1][0, 149]) and (lse[1] == 64.0).all()
    assert (sums[1, 0, :149] == 0).all() and abs(float(sums[1, 0, 149]) - 2) <= 8 * U
    mean = c.rows[2][1][0].double().mean(0).cpu()
    a = c.rows[2][1][0].double().abs().mean(0).cpu()
    _near(o[2, 0], mean, _half(BF) * (mean.abs() + 200 * U * a) + 200 * U * a, "equal lowest scores")


@pytest.mark.parametrize("page,dtype,D", [(16, BF, 64), (5, BF, 64), (64, HF, 64), (7, HF, 128), (128, BF, 128), (3, BF, 40)])
def test_decode_paged_infinite_values_and_nan_queries(page, dtype, D):
    """An infinite value with weight makes its dim infinite; a query of NaN makes its own head NaN.  The other dims, and
    the other heads of the key-value head, keep their accuracy."""
    g = _gen(20 + page)
    H, H_kv, L = 8, 2, 700
    c = Paged(g, [L, L, 0], H_kv, D, page, dtype, sigma=0.5)
    q = _randn((3, H, D), g, dtype)
    rows = [[t.clone() for t in r] for r in c.rows]
    for j, d, x in ((3, 7, INF), (600, 9, -INF), (650, 9, -INF)):
        rows[0][1][1, j, d] = x
        c.row(c.v, 0, j)[1, d] = x
    q[1, 2, 5] = NAN
    o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, return_lse=True)
    torch.cuda.synchronize()
    finite = rows[0][1].clone()
    finite[torch.isinf(finite)] = 0
    ro, rl, _, eo, el, _ = attend(q[0], rows[0][0], finite, D ** -0.5)
    assert (o[0, 4:, 7] == INF).all() and (o[0, 4:, 9] == -INF).all()
    got = o[0].clone()
    got[4:, 7], got[4:, 9] = ro[4:, 7].to(got), ro[4:, 9].to(got)
    _near(got, ro, eo + _half(dtype) * (ro.abs() + eo), "beside infinite values")
    _near(lse[0], rl, el, "lse")
    assert torch.isnan(o[1, 2]).all() and torch.isnan(lse[1, 2])
    clean = q[1].clone()
    clean[2] = 0
    ro, rl, _, eo, el, _ = attend(clean, *rows[1], D ** -0.5)
    others = [h for h in range(H) if h != 2]
    _near(o[1, others], ro[others], (eo + _half(dtype) * (ro.abs() + eo))[others], "beside a head of NaN")
    _near(lse[1, others], rl[others], el[others], "lse")
    assert (o[2] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_paged_many_small_weights(dtype):
    """20000 rows of weight e^-17.4 beside one of weight 1, whose values are 0: fp16's smallest number is 6e-8, these
    weights 3e-8.  A weight below 2^-24 is kept to 2^-38 of the largest."""
    g = _gen(31)
    D, L, page = 64, 20000, 64
    c = Paged(g, [L], 1, D, page, dtype)
    (k, v), = c.rows
    k.zero_()
    k[0, 1:, 0] = -17.4
    v.add_(1.0)
    v[0, 0] = 0
    for j in range(0, L, page):
        m = min(page, L - j)
        c.k[int(c.table[0, j // page]), :, :m] = k[:, j:j + m]
        c.v[int(c.table[0, j // page]), :, :m] = v[:, j:j + m]
    q = torch.zeros(1, 1, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    ws = torch.empty(0, dtype=torch.uint8, device=DEV)   # (not divided: a quarter of the rows beside the first)
    o = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, softmax_scale=1.0, workspace=ws)
    ro, _, _, eo, _, _ = attend(q[0], k, v, 1.0)
    small = 2.0 ** -38 * v[0].double().abs().sum(0).cpu()
    _near(o[0], ro, eo + small + _half(dtype) * (ro.abs() + eo + small) + 2.0 ** -25, "o")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_paged_large_scores(dtype):
    """Scores near 2^23, where float32 holds integers only: a later row passes the first ones by 7, 2.1 with the scale.  The scores
    are exact, and so are their differences, which the weights come from: (L + 32) u for their sums, 2^-16 for the
    weights' own bits."""
    g = _gen(33)
    D, L, page = 64, 300, 16
    c = Paged(g, [L], 1, D, page, dtype)
    (k, v), = c.rows
    k.zero_()
    k[0, :, 0] = 256
    k[0, 128, 1] = 7
    for j in range(0, L, page):
        c.k[int(c.table[0, j // page]), :, :min(page, L - j)] = k[:, j:j + page]
    q = torch.zeros(1, 1, D, dtype=dtype, device=DEV)
    q[..., 0], q[..., 1] = 32768, 1
    o = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, softmax_scale=0.3)
    p = torch.softmax(k[0, :, 1].double().cpu() * 0.3, 0)
    vv = v[0].double().cpu()
    ro, eo = (p @ vv)[None], (((L + 32) * U + 2.0 ** -16) * (p @ vv.abs()))[None]
    _near(o[0], ro, eo + _half(dtype) * (ro.abs() + eo), "o")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("L,at", [(3, (0, 1, 2)), (300, (7, 40, 290)), (2500, (2499, 0, 1300))])
def test_decode_paged_weights_keep_their_bits(dtype, L, at):
    """Two rows of weight 1 whose values are minus the first and second 16-bit part of a third row's weight p, and that row
    with the value 1: the output is what two parts leave of p, over 2 + p.  (The other rows weigh e^-256.)  An exponential
    is off by 2 u of itself, its argument by another, and the sums of six products of at most 1 by 2 u each: 16 u in all."""
    g = _gen(35)
    H, D, page = 16, 64, 16
    c = Paged(g, [L], H, D, page, dtype)
    (k, v), = c.rows
    q = torch.zeros(1, H, D, dtype=dtype, device=DEV)
    q[0, :, 0] = (0.05 + 0.6 * torch.rand(H, generator=g)).to(dtype).to(DEV)
    q[..., 1] = 1
    p = torch.exp(-q[0, :, 0].double())
    hi = p.to(dtype)
    lo = (p - hi.double()).to(dtype)
    k.zero_()
    k[..., 1] = -256
    k[:, at, 1] = 0
    k[:, at[2], 0] = -1
    v[:, at[0]], v[:, at[1]], v[:, at[2]] = -hi[:, None], -lo[:, None], 1
    for j in range(0, L, page):
        m, pid = min(page, L - j), int(c.table[0, j // page])
        c.k[pid, :, :m], c.v[pid, :, :m] = k[:, j:j + m], v[:, j:j + m]
    o = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, softmax_scale=1.0)
    ro = ((p - hi.double() - lo.double()) / (2 + p)).cpu()[:, None].expand(H, D)
    eo = (16 * U / (2 + p)).cpu()[:, None]
    _near(o[0], ro, eo + _half(dtype) * (ro.abs() + eo) + 2.0 ** -25, "o")


def test_decode_paged_divides_more_than_64_sequences():
    """The division of the work takes lengths 64 at a time."""
    g = _gen(32)
    B, H, D, page = 150, 1, 64, 32
    lens = torch.randint(0, 700, (B,), generator=g).tolist()
    lens[3], lens[70], lens[149], lens[64], lens[127] = 5000, 3000, 2500, 0, 1
    c = Paged(g, lens, H, D, page, BF, spare=1)
    q, kn, vn = (_randn((B, H, D), g, BF) for _ in range(3))
    assert _C.decode_paged_workspace(B, H, H, page, c.table.shape[1], D, False) > 0
    sums = torch.zeros(B, H, c.table.shape[1] * page, device=DEV)
    o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, return_lse=True, key_weights=sums)
    torch.cuda.synchronize()
    for b in range(B):
        k, v = (torch.cat([t, n[b][:, None]], 1) for t, n in zip(c.rows[b], (kn, vn)))
        ro, rl, w, eo, el, ew = attend(q[b], k, v, D ** -0.5)
        for got, want, bound in ((o[b], ro, eo + _half(BF) * (ro.abs() + eo)), (lse[b], rl, el),
                                 (sums[b, :, :lens[b] + 1], w, ew + 2 * U * w)):
            assert ((got.double().cpu() - want).abs() <= bound).all(), (b, lens[b])


def test_decode_paged_many_units_and_one_long_sequence():
    """More units than four a CU, one sequence of 20000 rows among short ones, whose weights are summed too."""
    g = _gen(34)
    B, H, D, page = 130, 8, 64, 64
    lens = torch.randint(0, 60, (B,), generator=g).tolist()
    lens[77] = 20000
    c = Paged(g, lens, H, D, page, BF, spare=1)
    q, kn, vn = (_randn((B, H, D), g, BF) for _ in range(3))
    sums = torch.zeros(B, H, c.table.shape[1] * page, device=DEV)
    o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, return_lse=True, key_weights=sums)
    torch.cuda.synchronize()
    for b in (0, 1, 76, 77, 78, 129):
        k, v = (torch.cat([t, n[b][:, None]], 1) for t, n in zip(c.rows[b], (kn, vn)))
        ro, rl, w, eo, el, ew = attend(q[b], k, v, D ** -0.5)
        _near(o[b], ro, eo + _half(BF) * (ro.abs() + eo), f"o of {lens[b]}")
        _near(lse[b], rl, el, "lse")
        _near(sums[b, :, :lens[b] + 1], w, ew + 2 * U * w, "sums")


@pytest.mark.parametrize("H,H_kv,D,page,dtype,append", [
    (12, 12, 64, 16, BF, True), (8, 2, 128, 64, HF, True), (20, 1, 64, 10, BF, False), (4, 4, 40, 32, BF, True)])
def test_decode_paged_adds_key_weights(H, H_kv, D, page, dtype, append):
    g = _gen(7 + H)
    lens = [0, 1, 130, 1000, 17]
    c = Paged(g, lens, H_kv, D, page, dtype, spare=1 if append else 0)
    B, M = len(lens), c.table.shape[1]
    q = _randn((B, H, D), g, dtype)
    kn, vn = (_randn((B, H_kv, D), g, dtype), _randn((B, H_kv, D), g, dtype)) if append else (None, None)
    buf = torch.rand(H_kv, B, M * page + 5, generator=g).to(DEV)
    sums = buf.transpose(0, 1)
    before = sums.double().cpu()
    fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, key_weights=sums)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        k, v = c.rows[b]
        if append:
            k, v = torch.cat([k, kn[b][:, None]], 1), torch.cat([v, vn[b][:, None]], 1)
        _, _, w, _, _, ew = attend(q[b], k, v, D ** -0.5)
        want = before[b].clone()
        if append:
            want[:, n] = 0
        want[:, :w.shape[1]] += w
        bound = torch.zeros_like(want)
        bound[:, :w.shape[1]] = ew + (H // H_kv + 2) * U * want[:, :w.shape[1]]
        _near(sums[b], want, bound, f"L={n} sums")


@pytest.mark.parametrize("H,H_kv,D,page,dtype,append,lens", [
    (12, 12, 64, 16, BF, True, [3000, 0, 1, 1023, 1025]),
    (6, 2, 40, 100, HF, True, [5000, 130, 0]),
    (8, 2, 128, 64, BF, False, [4000, 128]),
    (16, 1, 64, 32, BF, True, [1000]),
    (2, 2, 64, 7, HF, True, [2300, 17]),        # a table of rows that are no multiple of 4
    (4, 4, 64, 64, BF, True, [9000, 2048, 40]),
    (16, 1, 64, 64, BF, True, [3000, 700]),
    (3, 3, 64, 64, BF, True, [4097]),
])
def test_decode_paged_adds_key_weights_of_long_caches(H, H_kv, D, page, dtype, append, lens):
    """The same where a cache is divided over workgroups, twice over; sums that were there stay under the new ones."""
    g = _gen(40 + H + page)
    c = Paged(g, lens, H_kv, D, page, dtype, spare=1 if append else 0)
    B, M = len(lens), c.table.shape[1]
    q = _randn((B, H, D), g, dtype)
    kn, vn = (_randn((B, H_kv, D), g, dtype), _randn((B, H_kv, D), g, dtype)) if append else (None, None)
    sums = torch.rand(B, H_kv, M * page, generator=g).to(DEV)
    before = sums.double().cpu()
    other = sums.clone()
    o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, key_weights=sums, return_lse=True)
    fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, key_weights=other)
    plain, plain_lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(sums, other) and torch.equal(o, plain) and torch.equal(lse, plain_lse)
    for b, n in enumerate(lens):
        k, v = c.rows[b]
        if append:
            k, v = torch.cat([k, kn[b][:, None]], 1), torch.cat([v, vn[b][:, None]], 1)
        _, _, w, _, _, ew = attend(q[b], k, v, D ** -0.5)
        want = before[b].clone()
        if append:
            want[:, n] = 0
        want[:, :w.shape[1]] += w
        bound = torch.zeros_like(want)
        bound[:, :w.shape[1]] = ew + (H // H_kv + 2) * U * want[:, :w.shape[1]]
        _near(sums[b], want, bound, f"L={n} sums")


@pytest.mark.parametrize("H,H_kv,L,page,append,dtype", [
    (2, 1, 300, 16, True, BF),       # added by the step's own workgroup
    (4, 2, 5000, 64, True, HF),      # by the one that joins a cache's parts
    (2, 1, 300, 7, False, BF),       # by a second kernel: a table of rows that are no multiple of 4,
    (20, 1, 500, 16, True, BF),      # two tiles of query heads,
    (3, 3, 9000, 64, True, HF),      # a long cache
])
def test_decode_paged_key_weights_of_large_scores(H, H_kv, L, page, append, dtype):
    """Scores near 2^23, exact, whose differences 0 to 12 are exact too: their weights are float32's to (L + 64) u, as the
    definition's exp(x_j) / sum exp(x_i) has them; scores and log-sum-exp by themselves are rounded to 0.25 here."""
    g = _gen(36 + L)
    c = Paged(g, [L], H_kv, 64, page, dtype, spare=1 if append else 0)
    (k, v), = c.rows
    k.zero_()
    k[..., 0] = 256
    k[..., 1] = torch.randint(0, 13, (H_kv, L), generator=g).to(dtype).to(DEV)
    for j in range(0, L, page):
        c.k[int(c.table[0, j // page]), :, :min(page, L - j)] = k[:, j:j + page]
    q = torch.zeros(1, H, 64, dtype=dtype, device=DEV)
    q[..., 0], q[..., 1] = 32768, 1
    kn = vn = None
    if append:
        kn, vn = torch.zeros(1, H_kv, 64, dtype=dtype, device=DEV), _randn((1, H_kv, 64), g, dtype)
        kn[..., 0], kn[..., 1] = 256, 9
        k = torch.cat([k, kn[0][:, None]], 1)
    sums = torch.zeros(1, H_kv, c.table.shape[1] * page, device=DEV)
    scale = 0.375
    fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, key_weights=sums, softmax_scale=scale)
    n = k.shape[1]
    want = H // H_kv * torch.softmax(k[..., 1].double().cpu() * scale, 1)
    _near(sums[0, :, :n], want, (L + 64) * U * want, "sums")
    assert (sums[0, :, n:] == 0).all()


def test_decode_paged_workspaces():
    """A workspace of any content and size: the division needs the whole of it, key weights refuse less."""
    g = _gen(8)
    H, D, page, lens = 4, 64, 64, [5000, 300]
    c = Paged(g, lens, H, D, page, BF)
    q = _randn((2, H, D), g, BF)
    args = (q, c.k, c.v, c.table, c.seqlens)
    M = c.table.shape[1]
    n = _C.decode_paged_workspace(2, H, H, page, M, D, True)
    assert 0 < _C.decode_paged_workspace(2, H, H, page, M, D, False) < n
    ref = fa.decode_paged(*args, return_lse=True)
    for fill in (0, 0x5A, 0xFF):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=DEV)
        for _ in range(2):
            o, lse = fa.decode_paged(*args, return_lse=True, workspace=ws)
            assert torch.equal(o, ref[0]) and torch.equal(lse, ref[1]), fill
    for size in (0, 4096):
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        o, lse = fa.decode_paged(*args, return_lse=True, workspace=ws)
        for b in range(2):
            ro, rl, _, eo, el, _ = attend(q[b], *c.rows[b], D ** -0.5)
            _near(o[b], ro, eo + _half(BF) * (ro.abs() + eo), f"workspace {size}")
            _near(lse[b], rl, el, "lse")
        with pytest.raises(RuntimeError, match="workspace too small"):
            fa.decode_paged(*args, key_weights=torch.zeros(2, H, M * page, device=DEV), workspace=ws)


def test_decode_paged_pools_past_32_bits():
    """Pages more than 2^32 bytes into the pool."""
    H_kv, page, D = 8, 64, 64
    P = 2 ** 32 // (H_kv * page * D * 2) + 40
    k, v = (torch.zeros(P, H_kv, page, D, dtype=BF, device=DEV) for _ in range(2))
    g = _gen(9)
    L = 1000
    ids = [P - 1 - 2 * i for i in range(-(-(L + 1) // page))]
    kk, vv = _randn((H_kv, L, D), g, BF), _randn((H_kv, L, D), g, BF)
    for j in range(0, L, page):
        m = min(page, L - j)
        k[ids[j // page], :, :m] = kk[:, j:j + m]
        v[ids[j // page], :, :m] = vv[:, j:j + m]
    q, kn, vn = _randn((1, H_kv, D), g, BF), _randn((1, H_kv, D), g, BF), _randn((1, H_kv, D), g, BF)
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    sl = torch.tensor([L], dtype=torch.int32, device=DEV)
    sums = torch.rand(1, H_kv, table.shape[1] * page, generator=g).to(DEV)
    o = fa.decode_paged(q, k, v, table, sl, kn, vn)
    new = torch.arange(0, 4, dtype=torch.int32, device=DEV)[None] * 2 + P - 38
    kept, _ = fa.evict(k, v, table, sl, sums, new, 200, recent=10)
    torch.cuda.synchronize()
    assert torch.equal(k[ids[L // page], :, L % page], kn[0]) and torch.equal(v[ids[L // page], :, L % page], vn[0])
    ro, _, _, eo, _, _ = attend(q[0], torch.cat([kk, kn[0][:, None]], 1), torch.cat([vv, vn[0][:, None]], 1), D ** -0.5)
    _near(o[0], ro, eo + _half(BF) * (ro.abs() + eo), "o")
    for h in range(H_kv):
        rows = kept[0, h].long()
        got = torch.cat([k[int(p), h] for p in new[0]])[:200]
        assert torch.equal(got, kk[h, rows])


def _weights_ref(q, k, lse, scale, causal, first):
    B, H, Nq, D = q.shape
    H_kv, Nk = k.shape[1:3]
    G = H // H_kv
    q, k, lse = q.double().cpu(), k.double().cpu(), lse.double().cpu()
    out, err = torch.zeros(B, H_kv, Nk, dtype=torch.float64), torch.zeros(B, H_kv, Nk, dtype=torch.float64)
    see = torch.arange(Nk) <= torch.arange(Nq)[:, None] + first if causal else torch.ones(Nq, Nk, dtype=torch.bool)
    for b in range(B):
        for h in range(H):
            x = scale * (q[b, h] @ k[b, h // G].T)
            z = lse[b, h][:, None]
            p = torch.where(see & (z > -INF), torch.exp(x - z), torch.zeros(()).double())
            X = scale * (q[b, h].abs() @ k[b, h // G].abs().T)
            e = (D + 4) * U * X + 4 * U * (x.abs() + z.abs())
            out[b, h // G] += p.sum(0)
            err[b, h // G] += torch.where(see & (z > -INF), p * 2.1 * e, torch.zeros(()).double()).sum(0)
    return out, err + (H // H_kv) * ((Nq + 16) * U * out + Nq * 2.0 ** -126)  # an exponential below 2^-126 is 0


@pytest.mark.parametrize("H,H_kv,Nq,Nk,D,dtype,causal,first", [
    (12, 12, 256, 256, 64, BF, True, 0),
    (4, 2, 1, 1, 64, BF, True, 0),
    (4, 4, 333, 333, 64, HF, True, 0),
    (8, 2, 64, 500, 128, HF, True, 436),
    (6, 2, 40, 500, 128, BF, True, 100),       # keys past every query
    (5, 5, 77, 130, 80, BF, False, 0),
    (3, 1, 129, 65, 40, HF, True, 7),          # queries past the keys
    (2, 2, 31, 33, 8, BF, True, 0),
    (16, 1, 5, 1000, 96, BF, True, 995),
])
def test_key_weights_match_64_bits(H, H_kv, Nq, Nk, D, dtype, causal, first):
    _say(f"weights H={H} H_kv={H_kv} Nq={Nq} Nk={Nk} D={D} {dtype} causal={causal} first={first}")
    g = _gen(H + Nk)
    B = 2
    q = _randn((B, Nq, H, D), g, dtype, 1.5).transpose(1, 2)
    k = _randn((B, Nk, H_kv, D), g, dtype, 1.5).transpose(1, 2)
    x = (q.float() @ k.float().repeat_interleave(H // H_kv, 1).transpose(-1, -2)) * D ** -0.5
    if causal:
        x.masked_fill_(torch.arange(Nk, device=DEV) > torch.arange(Nq, device=DEV)[:, None] + first, -INF)
    lse = torch.logsumexp(x, -1)
    wide = torch.full((B, H_kv, Nk + 7), 3.0, device=DEV)
    out = fa.key_weights(q, k, lse, first_query=first, causal=causal, out=wide[..., :Nk])
    torch.cuda.synchronize()
    ref, bound = _weights_ref(q, k, lse, D ** -0.5, causal, first)
    _near(out, ref, bound, "sums")
    assert (wide[..., Nk:] == 3).all()
    assert torch.equal(fa.key_weights(q, k, lse, first_query=first, causal=causal), out), "another run"


@pytest.mark.parametrize("B,H,H_kv,Nq,Nk,D,dtype,causal", [
    (1, 16, 1, 1000, 1000, 64, BF, True),
    (2, 24, 3, 700, 333, 128, HF, False),
    (1, 32, 4, 65, 300, 80, BF, True),
    (1, 3, 3, 2000, 129, 64, HF, True),      # the queries past the keys' positions see them all
    (1, 16, 1, 129, 2000, 40, BF, False),
])
def test_key_weights_divided_queries(B, H, H_kv, Nq, Nk, D, dtype, causal):
    """Few keys and many queries: the queries go to several workgroups, whose sums are added in order."""
    g = _gen(Nq + Nk)
    q, k = _randn((B, H, Nq, D), g, dtype), _randn((B, H_kv, Nk, D), g, dtype)
    G, scale = H // H_kv, D ** -0.5
    hide = (torch.arange(Nk)[None, :] > torch.arange(Nq)[:, None]) if causal else torch.zeros(Nq, Nk, dtype=torch.bool)
    lse, want, bound = torch.empty(B, H, Nq), torch.zeros(B, H_kv, Nk, dtype=torch.float64), torch.zeros(B, H_kv, Nk, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            qd, kd = q[b, h].double().cpu(), k[b, h // G].double().cpu()
            x = (scale * qd @ kd.T.contiguous()).masked_fill(hide, -INF)
            lse[b, h] = torch.logsumexp(x, 1).float()
            p = torch.exp(x - lse[b, h].double()[:, None])
            big = float((scale * qd.abs() @ kd.abs().T.contiguous()).max())
            e = 2.1 * ((D + 4) * U * big + 4 * U * (2 * big + float(lse[b, h].abs().max())))
            want[b, h // G] += p.sum(0)
            bound[b, h // G] += (e + (Nq * G + 80) * U) * p.sum(0)
    lse = lse.to(DEV)
    n = _C.key_weights_workspace(B, H, H_kv, Nq, Nk, causal)
    assert n > 0
    got = fa.key_weights(q, k, lse, causal=causal)
    _near(got, want, bound, "divided")
    _near(fa.key_weights(q, k, lse, causal=causal, workspace=torch.empty(64, dtype=torch.uint8, device=DEV)), want, bound, "whole")
    for fill in (0, 0x5A, 0xFF):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=DEV)
        for _ in range(3):
            assert torch.equal(fa.key_weights(q, k, lse, causal=causal, workspace=ws), got), fill
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        held = fa.key_weights(q, k, lse, causal=causal)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, got) and torch.equal(fa.key_weights(q, k, lse, causal=causal), got)


@pytest.mark.parametrize("H,H_kv,Nq,Nk,dtype,causal", [(4, 2, 200, 300, BF, True), (2, 2, 64, 64, HF, False),
                                                       (16, 1, 700, 700, BF, True)])
def test_key_weights_of_large_scores(H, H_kv, Nq, Nk, dtype, causal):
    """Scores near 2^23, which are exact, and a log-sum-exp near 786432 (scale 0.09375) or 838861 (0.1) as float32 holds it:
    exp(scale s - lse) is a function of those numbers, off by 4 u |scale s - lse| + 16 u of itself, sums by Nq u."""
    g = _gen(37)
    for scale in (0.09375, float(np.float32(0.1))):
        q, k = (torch.zeros(1, h, n, 64, dtype=dtype, device=DEV) for h, n in ((H, Nq), (H_kv, Nk)))
        q[..., 0], q[..., 1] = 32768, 1
        k[..., 0] = 256
        k[..., 1] = torch.randint(0, 13, (1, H_kv, Nk), generator=g).to(dtype).to(DEV)
        x = scale * (2.0 ** 23 + k[..., 1].double().cpu())
        lse = (torch.logsumexp(x, -1).repeat_interleave(H // H_kv, 1)[..., None] + torch.rand(1, H, Nq, generator=g)).float()
        d = x.repeat_interleave(H // H_kv, 1)[:, :, None] - lse.double()[..., None]
        see = torch.arange(Nk) <= torch.arange(Nq)[:, None] if causal else torch.ones(Nq, Nk, dtype=torch.bool)
        p = torch.where(see, torch.exp(d), 0.0)
        fold = lambda t: t.view(1, H_kv, -1, Nk).sum(2)  # noqa: E731
        want = fold(p)
        bound = fold(p * (4 * U * d.abs() + 16 * U)) + H // H_kv * Nq * U * want
        _near(fa.key_weights(q, k, lse.to(DEV), softmax_scale=scale, causal=causal), want, bound, f"scale {scale}")


def test_key_weights_of_hidden_and_empty_rows():
    """Keys that no query sees get 0 whatever they hold; a query whose lse is -inf adds nothing; NaN in a query
    reaches only the keys it sees; no queries at all give zeros."""
    g = _gen(12)
    q, k = _randn((1, 2, 100, 64), g, BF), _randn((1, 2, 300, 64), g, BF)
    x = (q.float() @ k.float().transpose(-1, -2)) / 8
    x.masked_fill_(torch.arange(300, device=DEV) > torch.arange(100, device=DEV)[:, None], -INF)
    lse = torch.logsumexp(x, -1)
    k[:, :, 100:] = NAN
    lse[0, 0, 40] = -INF
    out = fa.key_weights(q, k, lse)
    ref, bound = _weights_ref(q, torch.nan_to_num(k), lse, 0.125, True, 0)
    assert (out[:, :, 100:] == 0).all()
    _near(out, ref, bound + 1e-300, "sums")
    q2 = q.clone()
    q2[0, 1, 70] = NAN
    out2 = fa.key_weights(q2, k, lse)
    assert torch.isnan(out2[0, 1, :71]).all() and torch.equal(out2[0, 1, 71:], out[0, 1, 71:])
    assert torch.equal(out2[0, 0], out[0, 0])
    assert (fa.key_weights(q[:, :, :0], k, lse[:, :, :0]) == 0).all()
    # The weights of a row sum to 1.
    assert abs(float(out[0, 1].double().sum()) - 100) <= 100 * 300 * U * 8


def _evict_ref(w, n, budget, recent):
    """Kept rows (ascending) of one head: w (N,) float32."""
    count, tail = min(n, budget), min(n, recent)
    w = w[:n - tail].double().cpu().numpy() + 0.0
    nan = np.isnan(w)
    best = np.lexsort((np.arange(len(w)), np.where(nan, 0, -w), nan))[:count - tail]
    return np.sort(np.concatenate([best, np.arange(n - tail, n)])).astype(np.int64)


@pytest.mark.parametrize("H_kv,D,page,lens,budget,recent,dtype,rows_first", [
    (12, 64, 16, [300, 299, 1, 0, 130, 131], 130, 32, BF, False),
    (2, 128, 64, [5000, 4097, 4096], 4096, 100, HF, True),
    (3, 40, 7, [200, 50, 90], 64, 0, BF, False),
    (1, 8, 1, [40, 17], 9, 9, HF, False),
    (1, 64, 256, [40000, 9000], 777, 128, BF, False),
    (4, 96, 100, [1024, 600], 1, 1, BF, True),
    (2, 64, 16, [100, 20], 400, 5, BF, False),
])
def test_evict_keeps_the_largest_sums(H_kv, D, page, lens, budget, recent, dtype, rows_first):
    _say(f"evict H_kv={H_kv} D={D} page={page} lens={lens} budget={budget} recent={recent}")
    g = _gen(budget + D)
    B, M2 = len(lens), -(-budget // page)
    c = Paged(g, lens, H_kv, D, page, dtype, rows_first=rows_first, extra=B * M2 + 2)
    new = torch.tensor(c.free[:B * M2], dtype=torch.int32, device=DEV).view(B, M2)
    w = torch.randint(0, 60, (B, H_kv, c.table.shape[1] * page), generator=g).float().to(DEV) / 8 - 1   # ties, -0
    w = torch.where(w == 0, -w, w)
    w[..., ::37] = 0.0
    w[..., 5::41] = NAN
    w[..., 7::43] = INF
    w[..., 8::47] = -INF
    k0, v0 = c.k.clone(), c.v.clone()
    kept, ws = fa.evict(c.k, c.v, c.table, c.seqlens, w, new, budget, recent=recent)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        for h in range(H_kv):
            ref = _evict_ref(w[b, h], n, budget, recent)
            m = len(ref)
            rows = torch.from_numpy(ref).to(DEV)
            assert torch.equal(kept[b, h, :m].long(), rows) and (kept[b, h, m:] == -1).all(), (b, h)
            assert torch.equal(ws[b, h, :m].view(torch.int32), w[b, h, rows].view(torch.int32))
            assert (ws[b, h, m:] == 0).all()
            to = torch.arange(m, device=DEV)
            at = new[b, to // page].long()
            k0[at, h, to % page] = c.rows[b][0][h, rows]
            v0[at, h, to % page] = c.rows[b][1][h, rows]
    assert torch.equal(c.k.contiguous().view(torch.int16), k0.contiguous().view(torch.int16)), "K pool"
    assert torch.equal(c.v.contiguous().view(torch.int16), v0.contiguous().view(torch.int16)), "V pool"


@pytest.mark.parametrize("L,budget", [(3000, 900), (70000, 40000)])
def test_evict_writes_sums_in_place(L, budget):
    g = _gen(13)
    page, H_kv = 64, 2
    M2 = -(-budget // page)
    c = Paged(g, [L], H_kv, 8, page, BF, extra=M2)
    new = torch.tensor([c.free], dtype=torch.int32, device=DEV)
    w = torch.rand(1, H_kv, c.table.shape[1] * page + 3, generator=g).to(DEV)
    kept, ws = fa.evict(c.k, c.v, c.table, c.seqlens, w.clone(), new, budget, recent=50)
    w2 = w.clone()
    kept2, ws2 = fa.evict(c.k, c.v, c.table, c.seqlens, w2, new, budget, recent=50, weights_out=w2)
    assert ws2 is w2 and torch.equal(kept2, kept) and torch.equal(w2[..., :budget], ws)
    for h in range(H_kv):
        assert np.array_equal(kept[0, h].cpu().numpy(), _evict_ref(w[0, h], L, budget, 50))


def test_evict_marks_bad_lengths_and_pages():
    g = _gen(14)
    c = Paged(g, [100, 100, 100, 100, 100], 2, 64, 16, BF, cols=8, extra=30)
    new = torch.tensor(c.free[:20], dtype=torch.int32, device=DEV).view(5, 4)
    table = c.table.clone()
    table[1, 6] = c.P
    new[2, 3] = -1
    sl = c.seqlens.clone()
    sl[3], sl[4] = -1, 8 * 16 + 1
    w = torch.rand(5, 2, 128, generator=g).to(DEV)
    k0 = c.k.clone()
    kept, ws = fa.evict(c.k, c.v, table, sl, w, new, 60, recent=4)
    torch.cuda.synchronize()
    assert (kept[1:] == -1).all() and torch.isnan(ws[1:]).all() and torch.isfinite(ws[0]).all()
    for h in range(2):
        rows = torch.from_numpy(_evict_ref(w[0, h], 100, 60, 4)).to(DEV)
        assert torch.equal(kept[0, h].long(), rows)
        to = torch.arange(60, device=DEV)
        k0[new[0, to // 16].long(), h, to % 16] = c.rows[0][0][h, rows]
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))


def test_evict_checks_pages_of_more_than_2_to_30_rows():
    """L + page passes 2^31: the page ids are checked all the same, and a good one's last rows are found."""
    page, L = 1200 * 10 ** 6, 1100 * 10 ** 6
    k = torch.empty(2, 1, page, 8, dtype=BF, device=DEV)
    w = torch.empty(1, 1, page, device=DEV)
    k[0, 0, L - 4:L] = _randn((4, 8), _gen(16), BF)
    w[0, 0, L - 4:L] = torch.arange(4, device=DEV).float()
    new = torch.ones(1, 1, dtype=torch.int32, device=DEV)
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    for pid in (2, -1):
        k[1, 0, :4] = 7
        kept, ws = fa.evict(k, k, new * pid, lens, w, new, 4, recent=4)
        assert (kept == -1).all() and torch.isnan(ws).all() and (k[1, 0, :4] == 7).all(), pid
    kept, ws = fa.evict(k, k, new * 0, lens, w, new, 4, recent=4)
    assert kept[0, 0].tolist() == list(range(L - 4, L)) and ws[0, 0].tolist() == [0, 1, 2, 3]
    assert torch.equal(k[1, 0, :4], k[0, 0, L - 4:L])


def _penalize_ref(x, tokens, lengths, rep, pres, freq, bias, allowed):
    B, V = x.shape
    x = x.double().cpu().numpy().copy()
    bound = np.abs(x) * 2
    col = lambda p, b: float(p[b]) if torch.is_tensor(p) else float(np.float32(p))  # noqa: E731
    for b in range(B):
        if tokens is not None:
            t = tokens[b].cpu().numpy()
            if lengths is not None:
                t = t[:max(0, int(lengths[b]))]
            n = np.bincount(t[(t >= 0) & (t < V)], minlength=V)
            s = n > 0
            r = col(rep, b)
            x[b] = np.where(s, np.where(x[b] > 0, x[b] / r, x[b] * r) - col(freq, b) * n - col(pres, b), x[b])
            bound[b] += np.abs(x[b]) + s * (abs(col(freq, b)) * n + abs(col(pres, b)))
        if bias is not None:
            y = (bias if bias.dim() == 1 else bias[b]).double().cpu().numpy()
            x[b] += y
            bound[b] += np.abs(y)
        if allowed is not None:
            a = (allowed if allowed.dim() == 1 else allowed[b]).cpu().numpy().view(np.uint8)
            off = np.unpackbits(a, bitorder="little")[:V] == 0
            x[b, off] = -INF
    return x, bound


@pytest.mark.parametrize("B,V,T,dtype,rows,ints,bias,allowed", [
    (1, 50257, 300, F32, False, torch.int64, None, None),
    (3, 50257, 1000, BF, True, torch.int64, "rows", "rows"),
    (5, 1000, 4097, HF, True, torch.int32, "shared", "shared"),
    (2, 33, 1, F32, True, torch.int32, "shared", "rows"),
    (4, 1, 9, F32, False, torch.int64, None, "rows"),
    (2, 4097, 0, BF, False, torch.int64, "rows", None),
    (70, 8193, 20, F32, True, torch.int64, None, "shared"),
])
def test_penalize_logits_matches_64_bits(B, V, T, dtype, rows, ints, bias, allowed):
    _say(f"logits B={B} V={V} T={T} {dtype}")
    g = _gen(V + B)
    x = _randn((B, V), g, dtype, 5.0)
    x[:, V // 3] = 0
    x[:, V // 2] = -INF
    tokens = (torch.rand(B, T, generator=g) ** 4 * (V + 2)).to(ints).to(DEV) - 1   # -1 and V among them
    rep, pres, freq, lengths = 1.3, 0.25, 0.125, None
    if rows:
        rep, pres, freq = (torch.rand(B, generator=g).to(DEV) + 0.5 for _ in range(3))
        lengths = torch.randint(-2, T + 5, (B,), generator=g, dtype=torch.int32).to(DEV)
    b = None if bias is None else _randn((V,) if bias == "shared" else (B, V), g, F32)
    W = -(-V // 32)
    a = None if allowed is None else torch.randint(-2 ** 31, 2 ** 31, (W,) if allowed == "shared" else (B, W),
                                                   generator=g).to(torch.int32).to(DEV)
    if a is not None:
        x[:, -1] = NAN   # a masked place may hold anything
        a[..., (V - 1) // 32] &= ~(1 << ((V - 1) % 32)) if (V - 1) % 32 != 31 else 0x7FFFFFFF
    y = fa.penalize_logits(x, tokens, lengths=lengths, repetition=rep, presence=pres, frequency=freq, bias=b, allowed=a)
    torch.cuda.synchronize()
    want, bound = _penalize_ref(torch.nan_to_num(x, nan=0.0, neginf=-INF), tokens, lengths, rep, pres, freq, b, a)
    got = y.double().cpu().numpy()
    assert y.dtype == dtype and np.array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    half, tiny = (_half(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps) if dtype != F32 else (0, 0)
    limit = 6 * U * bound[fin] + half * (np.abs(want[fin]) + 6 * U * bound[fin]) + tiny
    d = np.abs(got[fin] - want[fin])
    _say(f"  max off {d.max() if d.size else 0:.3e}")
    assert (d <= limit).all()
    # In place, with row strides.
    wide = torch.zeros(B, V + 3, dtype=dtype, device=DEV)
    wide[:, :V] = x
    z = fa.penalize_logits(wide[:, :V], tokens, lengths=lengths, repetition=rep, presence=pres, frequency=freq, bias=b,
                           allowed=a, out=wide[:, :V])
    assert z.data_ptr() == wide.data_ptr() and torch.equal(z, y) and (wide[:, V:] == 0).all()


def test_serving_operators_replay_from_graphs():
    """Two captured graphs and eager work in turn: every replay equals the eager result, bit for bit."""
    g = _gen(20)
    H, H_kv, D, page, lens = 8, 2, 64, 32, [900, 64, 3000]
    c = Paged(g, lens, H_kv, D, page, BF, spare=1, extra=3 * 16)
    new = torch.tensor(c.free, dtype=torch.int32, device=DEV).view(3, 16)
    q, kn, vn = (_randn((3, n, D), g, BF) for n in (H, H_kv, H_kv))
    w0 = torch.rand(3, H_kv, c.table.shape[1] * page, generator=g).to(DEV)
    pq, pk = _randn((1, H, 300, D), g, BF), _randn((1, H_kv, 300, D), g, BF)
    pl = torch.full((1, H, 300), 5.0, device=DEV)
    logits, toks = _randn((3, 5000), g, F32), torch.randint(0, 5000, (3, 40), generator=g).to(DEV)
    w = w0.clone()

    def work():
        w.copy_(w0)
        o, lse = fa.decode_paged(q, c.k, c.v, c.table, c.seqlens, kn, vn, key_weights=w, return_lse=True)
        kept, ws = fa.evict(c.k, c.v, c.table, c.seqlens, w, new, 500, recent=40)
        return o, lse, kept, ws, fa.key_weights(pq, pk, pl), fa.penalize_logits(logits, toks, repetition=1.2)

    ref = [t.clone() for t in work()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            got = work()
        graphs.append((graph, got))
    torch.cuda.current_stream().wait_stream(side)
    for rep in range(3):
        for n, (graph, got) in enumerate(graphs):
            for t in got:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            _say(f"replay {rep} of graph {n}")
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), (rep, n)
        assert all(torch.equal(a, b) for a, b in zip(work(), ref)), f"eager {rep}"


def test_serving_operators_on_streams_of_their_own():
    """Different steps on two streams at once, each with its own workspace, equal to one after the other."""
    g = _gen(21)
    sets = []
    for lens, H, H_kv in (([4000, 100], 4, 4), ([2500], 16, 2)):
        c = Paged(g, lens, H_kv, 64, 16, BF)
        sets.append((c, _randn((len(lens), H, 64), g, BF)))
    refs = [fa.decode_paged(q, c.k, c.v, c.table, c.seqlens) for c, q in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        outs = []
        for s, (c, q) in zip(streams, sets):
            with torch.cuda.stream(s):
                outs.append([fa.decode_paged(q, c.k, c.v, c.table, c.seqlens) for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for got, r in zip(outs, refs) for o in got)


def test_threads_share_a_stream_and_its_workspace():
    """Steps of four threads on one stream, whose calls share one workspace: each gives what it gives by itself, key
    weights that a second kernel adds from scores in the workspace among them."""
    import threading

    g = _gen(22)
    sets = []
    for L, H, H_kv, page in ((9000, 3, 3, 64), (1500, 20, 1, 7)):
        c = Paged(g, [L], H_kv, 64, page, BF)
        sets.append((_randn((1, H, 64), g, BF), c.k, c.v, c.table, c.seqlens))

    def paged(n):
        w = torch.zeros(1, sets[n][1].shape[1], sets[n][3].shape[1] * sets[n][1].shape[2], device=DEV)
        return fa.decode_paged(*sets[n], key_weights=w), w

    step = [_randn((1, 4, 64), g, BF)] + [_randn((1, 4, 6000, 64), g, BF) for _ in range(2)]
    prompt = [_randn((1, h, 700, 64), g, BF) for h in (16, 1)] + [torch.full((1, 16, 700), 6.0, device=DEV)]
    assert _C.decode_workspace_size(1, 4, 6000, 64) > 0 and _C.key_weights_workspace(1, 16, 1, 700, 700, True) > 0
    calls = [lambda: paged(0), lambda: paged(1), lambda: (fa.decode(*step),), lambda: (fa.key_weights(*prompt),)]
    refs = [call() for call in calls]
    torch.cuda.synchronize()
    got, stream = [[] for _ in calls], torch.cuda.current_stream()

    def run(n):
        with torch.cuda.stream(stream):
            for _ in range(100):
                got[n].append(calls[n]())

    threads = [threading.Thread(target=run, args=(n,)) for n in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for n, ref in enumerate(refs):
        assert len(got[n]) == 100
        assert all(torch.equal(a, b) for outs in got[n] for a, b in zip(outs, ref)), n


def test_empty_calls():
    k = torch.zeros(2, 1, 16, 64, dtype=BF, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    o, lse = fa.decode_paged(torch.zeros(0, 4, 64, dtype=BF, device=DEV), k, k, torch.zeros(0, 3, **i32),
                             torch.zeros(0, **i32), return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    o, lse = fa.decode_paged(torch.zeros(2, 4, 64, dtype=BF, device=DEV), k, k, torch.zeros(2, 0, **i32),
                             torch.zeros(2, **i32), return_lse=True)
    assert (o == 0).all() and (lse == -INF).all()
    kept, ws = fa.evict(k, k, torch.zeros(2, 0, **i32), torch.zeros(2, **i32), torch.zeros(2, 1, 0, device=DEV),
                        torch.ones(2, 1, **i32), 5)
    assert (kept == -1).all() and (ws == 0).all()
    assert fa.penalize_logits(torch.zeros(0, 9, device=DEV)).shape == (0, 9)
    assert fa.penalize_logits(torch.zeros(3, 0, device=DEV)).shape == (3, 0)


def test_prompt_steps_and_cuts_run_together():
    """A paged cache as a generation uses it: the prompt's attention and key weights, steps that append and sum weights,
    cuts to the budget in between; against the same in 64 bits.  (Which rows a cut keeps is checked on the sums that the
    cache holds, which are themselves within their bound.)"""
    import model_inference as mi

    g = _gen(30)
    B, H, D, N, steps = 2, 3, 64, 150, 60
    cache = mi.PagedKVCache({"n_heads": H, "emb_dim": H * D, "n_layers": 1}, B, 256, DEV, page_size=16, budget=64, recent=20,
                            slack=17)
    q, k, v = (_randn((B, N, H, D), g, BF, 1.5) for _ in range(3))
    ctx = torch.empty(B, N, H, D, dtype=BF, device=DEV)
    cache.prompt(0, q, k, v, ctx)
    cache.advance(N)
    qd, kd = q.double().cpu(), k.double().cpu()
    rows = [[(k[b, :, :].transpose(0, 1).cpu(), v[b, :, :].transpose(0, 1).cpu()) for _ in (0,)][0] for b in range(B)]
    sums, err = torch.zeros(B, H, N, dtype=torch.float64), torch.zeros(B, H, N, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            x = (qd[b, :, h] @ kd[b, :, h].T) * D ** -0.5
            x.masked_fill_(torch.ones(N, N).triu(1).bool(), -INF)
            p = torch.softmax(x, 1)
            sums[b, h] = p.sum(0)
            X = (qd[b, :, h].abs() @ kd[b, :, h].abs().T * D ** -0.5).max()
            # The attention's lse is off by its scores' error and its bf16-weighted sum's 2^-8 at most.
            err[b, h] = sums[b, h] * (2.1 * ((D + 4) * U * X + 8 * U * x[x > -INF].abs().max()) + 2.0 ** -8 + N * U)
    for step in range(steps):
        assert torch.equal(cache.seqlens.cpu(), torch.full((B,), cache.length, dtype=torch.int32))
        assert (cache.positions == N + step).all()
        n = cache.length
        held = cache.weights[0][:, :, :n].double().cpu()
        assert ((held - sums).abs() <= err).all(), f"sums before step {step}"
        if cache.over():
            _say(f"step {step}: cut from {n} rows")
            w = cache.weights[0][:, :, :n].clone()
            cache.evict()
            assert cache.length == 64 and not cache.over()
            for b in range(B):
                for h in range(H):
                    keep = torch.from_numpy(_evict_ref(w[b, h], n, 64, 20))
                    sums[b, h, :64], err[b, h, :64] = sums[b, h, keep].clone(), err[b, h, keep].clone()
                    for t in rows[b]:
                        t[h, :64] = t[h, keep].clone()
            sums, err = sums[..., :64], err[..., :64]
            rows = [(kk[:, :64], vv[:, :64]) for kk, vv in rows]
        q1, k1, v1 = (_randn((B, H, D), g, BF, 1.5) for _ in range(3))
        o = cache.attend(0, q1, k1, v1)
        cache.advance(1)
        rows = [(torch.cat([rows[b][0], k1[b].cpu()[:, None]], 1), torch.cat([rows[b][1], v1[b].cpu()[:, None]], 1))
                for b in range(B)]
        zero = torch.zeros(B, H, 1, dtype=torch.float64)
        sums, err = torch.cat([sums, zero], 2), torch.cat([err, zero], 2)
        for b in range(B):
            ro, _, w, eo, _, ew = attend(q1[b], *rows[b], D ** -0.5)
            d = (o[b].double().cpu() - ro).abs()
            assert (d <= eo + _half(BF) * (ro.abs() + eo)).all(), step
            sums[b] += w
            err[b] += ew + 2 * U * sums[b]
    pages = torch.cat([cache.table.cpu().flatten(), torch.tensor(cache._free, dtype=torch.int32)])
    assert sorted(pages.tolist()) == list(range(cache.k[0].shape[0])), "every page is held or free once"
    cache.reset()
    assert cache.length == 0 and (cache.positions == 0).all() and cache.table.shape[1] == 16


def test_generation_with_paged_caches_and_penalties():
    """generate_cached over pages gives the logits of the contiguous cache (both bf16 attentions of one model); with a
    budget it runs past it; penalties forbid and demand tokens in every loop."""
    import model_inference as mi

    cfg = dict(mi.GPT_CONFIG_124M)
    cfg.update({"emb_dim": 256, "n_layers": 2, "n_heads": 4, "vocab_size": 1000, "context_length": 256, "drop_rate": 0.0,
                "qkv_bias": True, "impl_type": "hip"})
    model = mi.GPTModel(cfg).eval()
    mi.init_gpt2_weights(model, 5)
    model.to(DEV)
    small = {"n_heads": 4, "emb_dim": 256, "n_layers": 2}
    idx = torch.randint(0, 1000, (3, 90), generator=_gen(1)).to(DEV)
    tokens = torch.randint(0, 1000, (3, 20), generator=_gen(2)).to(DEV)
    caches = [mi.KVCache(small, 3, 128, DEV), mi.PagedKVCache(small, 3, 128, DEV, page_size=16),
              mi.PagedKVCache(small, 3, 128, DEV, page_size=48, budget=100, slack=28)]
    with torch.no_grad():
        got = [[model(idx, kv_cache=c)[:, -1]] + [model(tokens[:, i:i + 1], kv_cache=c)[:, -1] for i in range(20)]
               for c in caches]
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert (a - b).norm() / a.norm() <= 1e-2   # the gate of the cached path against the full forward
    cut = mi.PagedKVCache(small, 3, 200, DEV, page_size=16, budget=32, recent=8, slack=16)
    out = mi.generate_cached(model, idx, 100, 256, temperature=0.0, cache=cut)
    assert out.shape == (3, 190) and cut.length <= 48 and int(cut.positions[0]) == 189
    again = mi.generate_cached(model, idx, 100, 256, temperature=0.0, cache=cut)
    assert torch.equal(out, again)
    with pytest.raises(ValueError, match="shorter than prompt"):
        mi.generate_cached(model, idx, 111, 256, cache=cut)
    with pytest.raises(ValueError, match="for 3 sequences"):
        mi.generate_cached(model, idx[:1], 5, 256, cache=cut)
    # Only even tokens, none twice.
    even = torch.full((32,), 0x55555555, dtype=torch.int32, device=DEV)
    loops = (lambda p: mi.generate(model, idx, 12, 256, temperature=0.0, penalties=p),
             lambda p: mi.generate_cached(model, idx, 12, 256, temperature=0.0, penalties=p),
             lambda p: mi.generate_graphed(model, idx, 12, 256, temperature=0.0, penalties=p))
    for loop in loops:
        new = loop(mi.LogitPenalties(presence=1e4, allowed=even))[:, 90:]
        assert (new % 2 == 0).all()
        for b in range(3):
            assert len(set(new[b].tolist())) == 12 and not set(new[b].tolist()) & set(idx[b].tolist())
        bias = torch.zeros(1000, device=DEV)
        bias[77] = 1e4
        assert (loop(mi.LogitPenalties(bias=bias))[:, 90:] == 77).all()
