"""Attention of several rows over a paged cache (custom_flash_attn.attend_paged, decode_shared) against softmax in 64 bits
on the same inputs (needs a GPU).

Tolerances count roundings, u = 2^-24 for float32 and half = torch.finfo(type).eps / 2 for one rounding to the output's
type, as worst cases of the sums:
  * a score less its row's offset is a float32 sum of D exact products and the offset, off by (D + 5) u (2 X + 10) at most:
    X is the row's largest scale * sum |q_d k_d|, and the offset (scaled) is a score of the row, so within X, less 13 ln 2 or
    0; scale, log2 e and their product add 4 u (|x| + |lse|).  Together ex.
  * a weight relative to its row's sum is off by twice e^ex - 1, at most 4.2 ex; sums of L terms by (L + 16) u.
  * the weights' rounding for the product with V: with up to 64 rows a key-value head (tokens, or a group's sequences, times
    the query heads it is shared by) two parts, 2^-16 (bf16: cut off at 2^-7,
    the rest rounded) or 2^-22 (fp16) of each; with more rows one rounding, half, of each and of their sum: 2 half.  fp16 keeps
    weights to 2^-38 of the largest."""
import math
import sys

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


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _bits(t):
    return t.contiguous().view(torch.int16)


class Pool:
    """Pages dealt in random order to texts of given rows; what no text may see is NaN."""

    def __init__(self, g, H_kv, D, page, dtype, pages, rows_first=False):
        shape = (pages, page, H_kv, D) if rows_first else (pages, H_kv, page, D)
        self.k, self.v = (torch.full(shape, NAN, dtype=dtype, device=DEV) for _ in range(2))
        if rows_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.g, self.page, self.H_kv, self.D, self.dtype, self.P = g, page, H_kv, D, dtype, pages
        self.free = torch.randperm(pages, generator=g).tolist()

    def table(self, rows, spare=0):
        """Tables for texts of `rows` (and `spare` more) rows, absent pages far outside the pool."""
        need = [-(-(n + spare) // self.page) for n in rows]
        t = torch.full((len(rows), max(max(need), 1)), 2 ** 31 - 9, dtype=torch.int32)
        for b, n in enumerate(need):
            t[b, :n] = torch.tensor([self.free.pop() for _ in range(n)], dtype=torch.int32)
        return t

    def put(self, ids, k, v):
        """Rows k, v (H_kv, n, D) from the first of the text's on."""
        for j in range(0, k.shape[1], self.page):
            m = min(self.page, k.shape[1] - j)
            self.k[int(ids[j // self.page]), :, :m] = k[:, j:j + m]
            self.v[int(ids[j // self.page]), :, :m] = v[:, j:j + m]

    def texts(self, rows, sigma, spare=0):
        """A table and the texts' (k, v), in their pages."""
        table, texts = self.table(rows, spare), []
        for b, n in enumerate(rows):
            k, v = _randn((self.H_kv, n, self.D), self.g, self.dtype, sigma), _randn((self.H_kv, n, self.D), self.g, self.dtype)
            self.put(table[b], k, v)
            texts.append((k, v))
        return table, texts


def attend(q, k, v, seen, scale, dtype, rounded):
    """q (H, N, D) over k, v (H_kv, L, D) in 64 bits, row i of N seeing the first seen[i] keys: o, lse and the bounds of
    their errors (o's before its rounding)."""
    (H, N, _), (H_kv, L, _) = q.shape, k.shape
    q, k, v = (t.detach().double().to(DEV) for t in (q, k, v))
    hide = torch.arange(L, device=DEV)[None] >= torch.as_tensor(seen, device=DEV)[:, None]
    o, lse, eo, el = (torch.zeros(s, dtype=torch.float64, device=DEV) for s in ((*q.shape,), (H, N), (*q.shape,), (H, N)))
    w = 2 * _half(dtype) if rounded else {BF: 2.0 ** -16, HF: 2.0 ** -22}[dtype]
    for h in range(H):
        kk, vv = k[h * H_kv // H], v[h * H_kv // H]
        x = (scale * (q[h] @ kk.T)).masked_fill(hide, -INF)
        lse[h] = torch.logsumexp(x, 1)
        p = torch.softmax(x, 1).nan_to_num(0.0)
        vis = torch.where(hide.all(0)[:, None], 0.0, vv)
        o[h] = p @ vis
        X = (scale * (q[h].abs() @ kk.abs().T)).masked_fill(hide, 0.0).amax(1) if L else torch.zeros(N, device=DEV)
        top = x.masked_fill(hide, 0.0).abs().amax(1) if L else X
        fin = lse[h].nan_to_num(0.0, 0.0, 0.0).abs()
        ex = (q.shape[2] + 5) * U * (2 * X + 10) + 4 * U * (top + fin)
        el[h] = ex + (L + 16) * U + 2 * U * fin
        eo[h] = (4.2 * ex + (L + 16) * U + w)[:, None] * (p @ vis.abs()) + (2.0 ** -38 * vis.abs().sum(0) if dtype == HF else 0.0)
    return o.cpu(), lse.cpu(), eo.cpu(), el.cpu()


def _near(got, want, bound, what):
    got = got.double().cpu()
    assert torch.equal(torch.isneginf(got), torch.isneginf(want)), what
    fin = ~torch.isneginf(want)
    d = (got - want).abs()[fin]
    room = bound[fin]
    worst = float((d / room.clamp(min=1e-300)).max()) if d.numel() else 0.0
    _say(f"  {what}: max off {float(d.max()) if d.numel() else 0:.3e}, at most {worst:.2f} of its bound")
    assert torch.isfinite(got[fin]).all() and (d <= room).all(), what


def _near_o(got, want, bound, dtype, what):
    _near(got, want, bound + _half(dtype) * (want.abs() + bound) + (2.0 ** -25 if dtype == HF else 0.0), what)


def _run_attend(H, H_kv, D, page, dtype, N, held, new, causal=True, rows_first=False, sigma=1.5, workspace=None, seed=0):
    g = _gen(seed + H * 1000 + D + page + N)
    total = [h + n if causal else h for h, n in zip(held, new)]
    pool = Pool(g, H_kv, D, page, dtype, sum(-(-t // page) for t in total) + 3, rows_first)
    table, texts = pool.texts(total, sigma)
    q = _randn((len(held), N, H, D), g, dtype, sigma).transpose(1, 2)
    ragged = any(n != N for n in new)
    o, lse = fa.attend_paged(q, pool.k, pool.v, table.to(DEV), _i32(held), lengths=_i32(new) if ragged else None, causal=causal,
                             return_lse=True, workspace=workspace)
    torch.cuda.synchronize()
    assert o.dtype == dtype and o.shape == q.shape and lse.shape == q.shape[:3]
    for b, (h, n) in enumerate(zip(held, new)):
        seen = [h + i + 1 if causal else h for i in range(n)]
        ro, rl, eo, el = attend(q[b, :, :n], *texts[b], seen, D ** -0.5, dtype, N * H // H_kv > 64)
        _near_o(o[b, :, :n], ro, eo, dtype, f"held={h} new={n} o")
        _near(lse[b, :, :n], rl, el, f"held={h} new={n} lse")
        assert (o[b, :, n:] == 0).all() and (lse[b, :, n:] == -INF).all()
    return o, lse


HELD = [0, 1, 15, 17, 128, 700, 2500]


@pytest.mark.parametrize("H,H_kv,D,page,dtype,N,causal,rows_first", [
    (12, 12, 64, 16, BF, 4, True, False),
    (12, 12, 64, 64, BF, 33, True, False),
    (12, 12, 64, 64, BF, 130, True, True),
    (8, 2, 128, 128, HF, 5, True, True),
    (8, 2, 128, 48, HF, 16, True, False),
    (8, 2, 128, 128, BF, 70, True, False),
    (8, 2, 128, 32, HF, 200, True, True),
    (6, 3, 40, 7, BF, 20, True, False),
    (4, 4, 64, 100, HF, 150, True, False),
    (3, 1, 80, 1, BF, 40, True, True),
    (24, 1, 96, 8, HF, 3, True, False),
    (5, 5, 8, 24, BF, 1, True, False),
    (16, 1, 128, 33, BF, 6, True, False),
    (4, 2, 128, 20, HF, 65, True, False),
    (12, 12, 64, 16, HF, 7, False, False),
    (8, 2, 128, 64, BF, 90, False, True),
    (6, 2, 72, 5, HF, 300, False, False),
])
@pytest.mark.parametrize("ragged", [False, True])
def test_attend_paged_matches_64_bits(H, H_kv, D, page, dtype, N, causal, rows_first, ragged):
    _say(f"attend H={H},{H_kv} D={D} page={page} {dtype} N={N} causal={causal} ragged={ragged}")
    new = [N, 0, N, 1, N // 2, N, max(N - 1, 0)] if ragged else [N] * 7
    _run_attend(H, H_kv, D, page, dtype, N, HELD, new, causal, rows_first)


@pytest.mark.parametrize("N", [1, 3, 40, 200])
@pytest.mark.parametrize("page,dtype,D", [(64, BF, 64), (16, HF, 128), (50, BF, 128)])
def test_attend_paged_divided(N, page, dtype, D):
    """One long text: its rows divided over workgroups, with the library's workspace, none, and one of the size asked for."""
    held, H, H_kv = 9001, 8, 2
    M = -(-(held + N) // page)
    nbytes = _C.attend_workspace(1, H, H_kv, N, page, M, D)
    assert nbytes > 0
    a = _run_attend(H, H_kv, D, page, dtype, N, [held], [N])
    b = _run_attend(H, H_kv, D, page, dtype, N, [held], [N], workspace=torch.empty(0, dtype=torch.uint8, device=DEV))
    ws = torch.full((nbytes + 64,), 255, dtype=torch.uint8, device=DEV)
    c = _run_attend(H, H_kv, D, page, dtype, N, [held], [N], workspace=ws[:nbytes])
    assert (ws[nbytes:] == 255).all()
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    assert (a[1] - b[1]).abs().max() <= 1e-4


def test_attend_paged_equals_attention_of_a_contiguous_prompt():
    g = _gen(4)
    B, H, N, D = 2, 12, 700, 64
    q, k, v = (_randn((B, H, N, D), g, BF) for _ in range(3))
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
    o, lse = fa.attend_paged(q, k, v, table, _i32([0, 0]), return_lse=True)
    o2, lse2 = fa.attention(q, k, v, return_lse=True)
    assert (o.double() - o2.double()).abs().max() <= 4 * _half(BF) * v.abs().max().double()
    assert (lse - lse2).abs().max() <= 1e-4


def test_attend_paged_takes_strides_out_and_scale():
    g = _gen(5)
    H, H_kv, D, N, page = 8, 4, 64, 50, 32
    for N in (3, 50):
        pool = Pool(g, H_kv, D, page, BF, 40)
        table, texts = pool.texts([70 + N, 300 + N], 1.0)
        wide = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        q = _randn((2, N, H, D + 24), g, BF)[..., 8:D + 8].transpose(1, 2)
        out = torch.full((N, H, 2, D + 8), 3.0, dtype=BF, device=DEV)
        got, lse = fa.attend_paged(q, pool.k, pool.v, wide[:, :20], _i32([70, 300]), lengths=_i32([N, N - 2]), softmax_scale=0.3,
                                   out=out.permute(2, 1, 0, 3)[..., :D], return_lse=True)
        assert got.data_ptr() == out.data_ptr()
        for b, n in ((0, N), (1, N - 2)):
            seen = [(70, 300)[b] + i + 1 for i in range(n)]
            ro, rl, eo, el = attend(q[b, :, :n], *texts[b], seen, 0.3, BF, N * 2 > 64)
            _near_o(got[b, :, :n], ro, eo, BF, f"b={b}")
            _near(lse[b, :, :n], rl, el, "lse")
        assert (out[..., D:] == 3).all() and (got[1, :, N - 2:] == 3).all() and (lse[1, :, N - 2:] == -INF).all()


@pytest.mark.parametrize("N", [2, 40, 150])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("divided", [False, True])
def test_attend_paged_marks_bad_lengths_and_pages(N, page, divided):
    g = _gen(6)
    H, H_kv, D, rows = 4, 2, 64, 900
    pool = Pool(g, H_kv, D, page, BF, 6 * 60)
    held = [200, 600, 300, 100, 100, 100]
    table, texts = pool.texts([h + N for h in held], 1.0)
    wide = torch.full((6, rows // page), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table[:, :rows // page]
    wide[1, 10] = pool.P                      # rows that every token sees
    wide[2, (300 + N - 1) // page] = -1       # rows that the last tokens see
    lens, lengths = _i32(held), _i32([N] * 6)
    lens[3] = -1
    lens[4] = rows - N + 1                    # one row too many
    lengths[5] = N + 1
    q = _randn((6, H, N, D), g, BF)
    ws = None if divided else torch.empty(0, dtype=torch.uint8, device=DEV)
    o, lse = fa.attend_paged(q, pool.k, pool.v, wide.to(DEV), lens, lengths=lengths, return_lse=True, workspace=ws)
    torch.cuda.synchronize()
    first_bad = (300 + N - 1) // page * page - 300   # of text 2: the first token that sees the page
    good = max(0, min(N, first_bad))
    _say(f"N={N} page={page}: {good} tokens of the third text are good")
    for b, n in ((0, N), (2, good)):
        ro, rl, eo, el = attend(q[b, :, :n], *texts[b], [held[b] + i + 1 for i in range(n)], D ** -0.5, BF, N * 2 > 64)
        _near_o(o[b, :, :n], ro, eo, BF, f"text {b}")
        _near(lse[b, :, :n], rl, el, "lse")
        assert torch.isnan(o[b, :, n:]).all() and torch.isnan(lse[b, :, n:]).all()
    for b in (1, 3, 4, 5):
        assert torch.isnan(o[b]).all() and torch.isnan(lse[b]).all()
    # Without causality the rows before the tokens are all: every page of text 2 that counts is good.
    o = fa.attend_paged(q[2:3], pool.k, pool.v, wide[2:3].to(DEV), _i32([200]), causal=False)
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("N,G", [(8, 2), (50, 1), (140, 1), (90, 2)])
@pytest.mark.parametrize("page,dtype,D", [(16, BF, 64), (12, HF, 64), (64, HF, 128), (64, BF, 128)])
def test_attend_paged_hidden_rows_and_infinite_values(N, G, page, dtype, D):
    """Keys and values of later tokens are NaN and infinite for the earlier ones, which do not see them; a value that is
    seen and infinite makes its dim infinite, and the rest keeps its accuracy."""
    g = _gen(7)
    H_kv, held = 2, 333
    pool = Pool(g, H_kv, D, page, dtype, 60)
    table, texts = pool.texts([held + N], 0.7)
    (k, v), = texts
    late = held + N // 2
    k[0, late], v[0, late + 1], v[1, late + 1, 3], v[1, 5, 9] = NAN, NAN, INF, -INF
    pool.put(table[0], k, v)
    q = _randn((1, H_kv * G, N, D), g, dtype, 0.7)
    o, lse = fa.attend_paged(q, pool.k, pool.v, table.to(DEV), _i32([held]), return_lse=True)
    torch.cuda.synchronize()
    clean_v = v.clone()
    clean_v[1, 5, 9] = 0
    n, rounded = N // 2, N * G > 64
    ro, rl, eo, el = attend(q[0, :, :n], k[:, :late], clean_v[:, :late], [held + i + 1 for i in range(n)], D ** -0.5, dtype, rounded)
    assert (o[0, G:, :, 9] == -INF).all()
    got = o[0, :, :n].clone()
    got[G:, :, 9] = ro[G:, :, 9].to(got)
    _near_o(got, ro, eo, dtype, "before the bad rows")
    _near(lse[0, :, :n], rl, el, "lse")
    assert torch.isnan(o[0, :G, n:]).all() and torch.isnan(lse[0, :G, n:]).all()
    # The other key-value head: from the next token on dim 3 is infinite, the others finite but dim 9.
    ro, rl, eo, el = attend(q[0, G:, :], k[1:], torch.where(torch.isfinite(v[1:]), v[1:], 0.0), [held + i + 1 for i in range(N)],
                            D ** -0.5, dtype, rounded)
    assert (o[0, G:, n + 1:, 3] == INF).all()
    dims = [d for d in range(D) if d not in (3, 9)]
    _near_o(o[0, G:][..., dims], ro[..., dims], eo[..., dims], dtype, "beside infinite values")
    _near(lse[0, G:], rl, el, "lse")


@pytest.mark.parametrize("N", [3, 60, 200])
def test_attend_paged_scores_of_minus_infinity_and_the_lowest(N):
    """Scores of -inf have weight 0, nothing else gives O = 0 and LSE = -inf; scores of the type's lowest value are finite
    and share the weight."""
    g = _gen(8)
    D, L, page = 64, 150, 16
    pool = Pool(g, 1, D, page, BF, 80)
    table, texts = pool.texts([L + N] * 3, 1.0)
    k = [t[0].clone() for t in texts]
    k[0][:] = -INF
    k[1][:, :149] = -INF
    k[1][:, 149] = 1.0
    k[1][:, 150:] = -INF
    k[2][:] = torch.finfo(BF).min / 64
    for b in range(3):
        pool.put(table[b], k[b], texts[b][1])
    q = torch.ones(3, 1, N, D, dtype=BF, device=DEV)
    o, lse = fa.attend_paged(q, pool.k, pool.v, table.to(DEV), _i32([L] * 3), return_lse=True, softmax_scale=1.0)
    assert (o[0] == 0).all() and (lse[0] == -INF).all()
    assert torch.equal(o[1, 0], texts[1][1][0, 149].expand(N, D)) and (lse[1] == 64.0).all()
    for i in (0, N - 1):
        v = texts[2][1][0, :L + i + 1].double().cpu()
        mean, a = v.mean(0), v.abs().mean(0)
        _near_o(o[2, 0, i], mean, ((L + N + 32) * U + 2 * _half(BF)) * a, BF, f"equal lowest scores, token {i}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N", [2, 100])
def test_attend_paged_large_scores_and_small_weights(dtype, N):
    """Scores near 2^23, where float32 holds integers only: exact, as are their differences; and 20000 rows of weight
    e^-17.4, below fp16's smallest number, beside one of weight 1 whose value is 0."""
    g = _gen(9)
    D, L, page = 64, 300, 16
    pool = Pool(g, 1, D, page, dtype, 60)
    table, texts = pool.texts([L + N], 1.0)
    (k, v), = texts
    k.zero_()
    k[0, :, 0] = 256
    k[0, 128, 1] = 7
    pool.put(table[0], k, v)
    q = torch.zeros(1, 1, N, D, dtype=dtype, device=DEV)
    q[..., 0], q[..., 1] = 32768, 1
    o = fa.attend_paged(q, pool.k, pool.v, table.to(DEV), _i32([L]), softmax_scale=0.3)
    w = 2 * _half(dtype) if N > 64 else 2.0 ** -16
    for i in (0, N - 1):
        p = torch.softmax(k[0, :L + i + 1, 1].double().cpu() * 0.3, 0)
        vv = v[0, :L + i + 1].double().cpu()
        # (2^-16 for the weights' own bits.)
        _near_o(o[0, 0, i], p @ vv, ((L + N + 32) * U + 2.0 ** -16 + w) * (p @ vv.abs()), dtype, f"token {i}")
    D, L, page = 64, 20000, 64
    pool = Pool(g, 1, D, page, dtype, 330)
    table, texts = pool.texts([L + N], 1.0)
    (k, v), = texts
    k.zero_()
    k[0, 1:, 0] = -17.4
    v.add_(1.0)
    v[0, 0] = 0
    pool.put(table[0], k, v)
    q = torch.zeros(1, 1, N, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    ws = torch.empty(0, dtype=torch.uint8, device=DEV)   # (not divided)
    o = fa.attend_paged(q, pool.k, pool.v, table.to(DEV), _i32([L]), softmax_scale=1.0, workspace=ws)
    ro, _, eo, _ = attend(q[0, :, :1], k, v, [L + 1], 1.0, dtype, N > 64)
    _near_o(o[0, :, :1], ro, eo, dtype, "small weights")


def test_attend_paged_empty_and_repeated():
    g = _gen(10)
    pool = Pool(g, 2, 64, 16, BF, 30)
    table, _ = pool.texts([100, 40], 1.0)
    t = table.to(DEV)
    for shape in ((0, 4, 5, 64), (2, 0, 5, 64), (2, 4, 0, 64)):
        q = torch.empty(shape, dtype=BF, device=DEV)
        assert fa.attend_paged(q, pool.k, pool.v, t[:shape[0]], _i32([90, 30])[:shape[0]]).shape == shape
    q = _randn((2, 4, 10, 64), g, BF)
    o, lse = fa.attend_paged(q, pool.k, pool.v, t[:, :0], _i32([0, 0]), causal=False, return_lse=True)   # no page at all
    assert (o == 0).all() and (lse == -INF).all()
    a = fa.attend_paged(q, pool.k, pool.v, t, _i32([90, 30]), return_lse=True)
    for _ in range(3):
        b = fa.attend_paged(q, pool.k, pool.v, t, _i32([90, 30]), return_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attend_paged_large_offsets():
    """A pool of more than 2^31 elements, and a page whose rows end past 2^31 bytes."""
    H_kv, page, D = 8, 65536, 128
    pool = torch.zeros((2, 40, H_kv, page, D), dtype=BF, device=DEV)
    g = _gen(11)
    n = page + 70
    k, v = _randn((H_kv, n, D), g, BF), _randn((H_kv, n, D), g, BF)
    for x, p in ((k, pool[0]), (v, pool[1])):
        p[39], p[38, :, :70] = x[:, :page], x[:, page:]
    table = _i32([[39, 38]])
    for N in (2, 130):
        q = _randn((1, 8, N, D), g, BF)
        o, lse = fa.attend_paged(q, pool[0], pool[1], table, _i32([n - N]), return_lse=True)
        seen = [n - N + i + 1 for i in range(N)]
        ro, rl, eo, el = attend(q[0, :, -1:], k, v, seen[-1:], D ** -0.5, BF, N > 64)
        _near_o(o[0, :, -1:], ro, eo, BF, f"N={N}")
        _near(lse[0, :, -1:], rl, el, "lse")


# ---------------------------------------------------------------------------------------
# Shared prefixes.


def _run_shared(H, H_kv, D, page, dtype, prefix, own, append, rows_first=False, sigma=1.5, seed=0):
    R, B = len(prefix), len(own)
    n, g = B // R, _gen(seed + H * 100 + D + page + B)
    pages = sum(-(-p // page) for p in prefix) + sum(-(-(o + 1) // page) for o in own) + 3
    pool = Pool(g, H_kv, D, page, dtype, pages, rows_first)
    ptable, before = pool.texts(prefix, sigma)
    table, texts = pool.texts(own, sigma, spare=1 if append else 0)
    q = _randn((B, H, D), g, dtype, sigma)
    kn, vn = (_randn((B, H_kv, D), g, dtype), _randn((B, H_kv, D), g, dtype)) if append else (None, None)
    k0, v0 = pool.k.clone(), pool.v.clone()
    o, lse = fa.decode_shared(q, pool.k, pool.v, ptable.to(DEV), _i32(prefix), table.to(DEV), _i32(own), kn, vn, return_lse=True)
    torch.cuda.synchronize()
    for b in range(B):
        k, v = (torch.cat([x, y], 1) for x, y in zip(before[b // n], texts[b]))
        if append:
            k, v = torch.cat([k, kn[b][:, None]], 1), torch.cat([v, vn[b][:, None]], 1)
            pid, off = int(table[b, own[b] // page]), own[b] % page
            k0[pid, :, off], v0[pid, :, off] = kn[b], vn[b]
        ro, rl, eo, el = attend(q[b][:, None], k, v, [k.shape[1]], D ** -0.5, dtype, n * H // H_kv > 64)
        _near_o(o[b][:, None], ro, eo, dtype, f"{b}: {prefix[b // n]} + {own[b]} o")
        _near(lse[b][:, None], rl, el, "lse")
    assert torch.equal(_bits(pool.k), _bits(k0)) and torch.equal(_bits(pool.v), _bits(v0)), "pool"


@pytest.mark.parametrize("H,H_kv,D,page,dtype,append,rows_first", [
    (12, 12, 64, 16, BF, True, False),
    (25, 25, 64, 64, BF, False, False),
    (8, 2, 128, 128, HF, True, True),
    (8, 2, 128, 48, BF, True, False),
    (4, 4, 64, 100, HF, False, False),
    (16, 1, 64, 1, BF, True, False),
    (40, 1, 96, 16, HF, True, False),      # more query heads than a tile has rows
    (6, 3, 80, 7, BF, True, True),
    (3, 3, 8, 24, HF, True, False),
    (6, 2, 40, 256, BF, True, False),
    (28, 4, 128, 33, HF, True, False),
])
@pytest.mark.parametrize("prefix,own", [
    ([700], [0, 5, 64, 301]),
    ([0, 33], [0, 16, 17, 1, 200, 2]),
    ([5000, 1], [3, 100, 31, 32]),
    ([64, 129, 1000], [40, 0, 700] * 4),
    ([333], [7 * i % 90 for i in range(40)]),
])
def test_decode_shared_matches_64_bits(H, H_kv, D, page, dtype, append, rows_first, prefix, own):
    _say(f"shared H={H},{H_kv} D={D} page={page} {dtype} prefix={prefix} own={own[:12]}")
    _run_shared(H, H_kv, D, page, dtype, prefix, own, append, rows_first)


def test_decode_shared_equals_decode_paged_of_the_same_pages():
    """A prefix of whole pages, named first in each sequence's own table, is what decode_paged reads for it."""
    g = _gen(31)
    H, H_kv, D, page, n = 8, 4, 64, 32, 6
    pool = Pool(g, H_kv, D, page, BF, 80)
    ptable, _ = pool.texts([320], 1.0)
    own = [0, 31, 32, 100, 5, 64]
    table, _ = pool.texts(own, 1.0, spare=1)
    q, kn, vn = _randn((n, H, D), g, BF), _randn((n, H_kv, D), g, BF), _randn((n, H_kv, D), g, BF)
    a, la = fa.decode_shared(q, pool.k, pool.v, ptable.to(DEV), _i32([320]), table.to(DEV), _i32(own), kn, vn, return_lse=True)
    whole = torch.cat([ptable.expand(n, -1), table], 1).to(DEV)
    b, lb = fa.decode_paged(q, pool.k, pool.v, whole, _i32([320 + x for x in own]), kn, vn, return_lse=True)
    assert (la - lb).abs().max() <= 1e-5
    assert (a.double() - b.double()).abs().max() <= 2 * _half(BF) * float(b.abs().max())


def test_decode_shared_marks_bad_lengths_and_pages():
    g = _gen(32)
    H, H_kv, D = 4, 2, 64
    for page in (16, 20):
        pool = Pool(g, H_kv, D, page, BF, 200)
        prefix, own = [100, 200, 300, 50], [10, 20, 30, 40, 50, 60, 70, 80]
        ptable, before = pool.texts(prefix, 1.0)
        table, texts = pool.texts(own, 1.0, spare=1)
        full = table.shape[1] * page
        pl, lens = _i32(prefix), _i32(own)
        pl[1] = ptable.shape[1] * page + 1     # group 1
        ptable[2, 3] = pool.P                  # group 2
        lens[1] = -1
        lens[6] = full                         # no room for the new row
        table[7, 80 // page] = -1              # the new row's page
        q, kn, vn = (_randn((8, n, D), g, BF) for n in (H, H_kv, H_kv))
        k0 = pool.k.clone()
        o, lse = fa.decode_shared(q, pool.k, pool.v, ptable.to(DEV), pl, table.to(DEV), lens, kn, vn, return_lse=True)
        torch.cuda.synchronize()
        _say(f"page {page}: nan {torch.isnan(lse).all(1).tolist()}")
        assert torch.isnan(o[1:]).all() and torch.isnan(lse[1:]).all()
        k, v = (torch.cat([x, y, z[0][:, None]], 1) for x, y, z in zip(before[0], texts[0], (kn, vn)))
        ro, rl, eo, el = attend(q[0][:, None], k, v, [111], D ** -0.5, BF, False)
        _near_o(o[0][:, None], ro, eo, BF, "good")
        for b in (0, 2, 3, 4, 5):
            k0[int(table[b, own[b] // page]), :, own[b] % page] = kn[b]
        assert torch.equal(_bits(pool.k), _bits(k0))


@pytest.mark.parametrize("n", [3, 50, 90])
def test_decode_shared_infinite_values_and_nan_queries(n):
    g = _gen(33)
    H, H_kv, D, page = 2, 1, 64, 16
    pool = Pool(g, H_kv, D, page, BF, 60 + n)
    ptable, before = pool.texts([500], 0.7)
    table, texts = pool.texts([9] * n, 0.7)
    k, v = before[0]
    v[0, 77, 5] = INF
    pool.put(ptable[0], k, v)
    texts[2][1][0, 3, 6] = -INF
    pool.put(table[2], *texts[2])
    q = _randn((n, H, D), g, BF)
    q[0, 1, 3] = NAN
    o, lse = fa.decode_shared(q, pool.k, pool.v, ptable.to(DEV), _i32([500]), table.to(DEV), _i32([9] * n), return_lse=True)
    assert torch.isnan(o[0, 1]).all() and torch.isnan(lse[0, 1])
    v[0, 77, 5] = 0
    texts[2][1][0, 3, 6] = 0
    for b, heads in ((0, [0]), (1, [0, 1]), (2, [0, 1]), (n - 1, [0, 1])):
        ro, rl, eo, el = attend(q[b, heads][:, None], torch.cat([k, texts[b][0]], 1), torch.cat([v, texts[b][1]], 1), [509],
                                D ** -0.5, BF, n * H // H_kv > 64)
        got = o[b, heads].clone()
        assert (got[:, 5] == INF).all() and (b != 2 or (got[:, 6] == -INF).all())
        bad = [5, 6] if b == 2 else [5]
        got[:, bad] = ro[:, 0, bad].to(got)
        _near_o(got[:, None], ro, eo, BF, f"sequence {b}")
        _near(lse[b, heads][:, None], rl, el, "lse")


def test_in_graphs_with_eager_calls_between():
    """append_paged, attend_paged and decode_shared captured on a side stream and replayed: two graphs whose workspaces
    are their own, eager calls between the replays, every replay against the eager result."""
    g = _gen(34)
    H, H_kv, D, page, B = 8, 2, 64, 16, 4
    pool = Pool(g, H_kv, D, page, BF, 700)
    ptable, _ = pool.texts([3000], 1.0)
    table, _ = pool.texts([1400, 800, 30, 1], 1.0, spare=200)
    pt, t, pl, start = ptable.to(DEV), table.to(DEV), _i32([3000]), _i32([1400, 800, 30, 1])
    rotary = fa.Rotary(64, device=DEV)
    lens = start.clone()
    q3, k3, v3 = _randn((B, H, 3, D), g, BF), _randn((B, H_kv, 3, D), g, BF), _randn((B, H_kv, 3, D), g, BF)
    q1, k1, v1 = _randn((B, H, D), g, BF), _randn((B, H_kv, D), g, BF), _randn((B, H_kv, D), g, BF)

    def chunk():
        q = fa.append_paged(k3, v3, pool.k, pool.v, t, lens, rotary=rotary, q=q3)
        return fa.attend_paged(q, pool.k, pool.v, t, lens, return_lse=True)

    def step():
        return fa.decode_shared(q1, pool.k, pool.v, pt, pl, t, lens, k1, v1, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for f in (chunk, step):
            f()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = f()
            graphs.append((graph, out, f))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        for x in (q3, k3, v3, q1, k1, v1):
            x.copy_(_randn(x.shape, g, BF))
        lens.copy_(start + 3 * i)   # (every row before them was appended)
        for graph, out, f in graphs:
            graph.replay()
            got = [x.clone() for x in out]
            want = f()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        torch.cuda.synchronize()


def _two_launch_calls(g):
    """Calls that keep parts in a workspace between two launches, on inputs of their own."""
    H, H_kv, D, page = 8, 2, 64, 16
    pool = Pool(g, H_kv, D, page, BF, 1300)
    long, _ = pool.texts([9000], 1.0)
    prefix, _ = pool.texts([3000], 1.0)
    own, _ = pool.texts([40, 0, 300, 17], 1.0, spare=1)
    other, _ = pool.texts([5000], 1.0)
    long, prefix, own, other = (x.to(DEV) for x in (long, prefix, own, other))
    q4, q60 = _randn((1, H, 4, D), g, BF), _randn((1, H, 60, D), g, BF)
    qs, q1 = _randn((4, H, D), g, BF), _randn((1, H, D), g, BF)
    lens = {n: _i32(n) for n in ((8996,), (8940,), (3000,), (40, 0, 300, 17), (5000,))}
    assert _C.attend_workspace(1, H, H_kv, 4, page, long.shape[1], D) > 0 and _C.attend_workspace(1, H, H_kv, 60, page, long.shape[1], D) > 0
    return [lambda: fa.attend_paged(q4, pool.k, pool.v, long, lens[(8996,)], return_lse=True),
            lambda: fa.attend_paged(q60, pool.k, pool.v, long, lens[(8940,)], return_lse=True),
            lambda: fa.decode_shared(qs, pool.k, pool.v, prefix, lens[(3000,)], own, lens[(40, 0, 300, 17)], return_lse=True),
            lambda: fa.decode_paged(q1, pool.k, pool.v, other, lens[(5000,)], return_lse=True)]


def test_threads_share_a_stream_and_its_workspace():
    """Calls of four threads on one stream, which share its workspace (a split decode step's among them): each gives what it
    gives by itself."""
    import threading

    calls = _two_launch_calls(_gen(36))
    refs = [call() for call in calls]
    torch.cuda.synchronize()
    got, stream = [[] for _ in calls], torch.cuda.current_stream()

    def run(n):
        with torch.cuda.stream(stream):
            for _ in range(60):
                got[n].append(calls[n]())

    threads = [threading.Thread(target=run, args=(n,)) for n in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for n, ref in enumerate(refs):
        assert len(got[n]) == 60
        assert all(torch.equal(a, b) for outs in got[n] for a, b in zip(outs, ref)), n


def test_two_streams_at_once():
    """The same calls on two streams, which may run at the same time, each with a workspace of its own."""
    calls = _two_launch_calls(_gen(37))
    refs = [call() for call in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(((i + k) % len(calls), calls[(i + k) % len(calls)]()))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for n, outs in got for a, b in zip(outs, refs[n]))


def test_prompt_in_chunks_then_samples_of_it():
    """The operators as a program runs them: two prompts go in by chunks of unequal lengths (rotated keys into the pages,
    attention over what is there), then three samples of each continue behind the shared prompt token by token; every
    output against plain attention over rotated keys and queries."""
    g = _gen(35)
    H, H_kv, D, page, R, n = 8, 2, 64, 16, 2, 3
    pool = Pool(g, H_kv, D, page, BF, 80)
    rotary = fa.Rotary(48, scaling="linear", factor=2.0, device=DEV)
    sizes = [150, 97]
    ptable = pool.table(sizes)
    k, v, q = (_randn((R, h, 150, D), g, BF) for h in (H_kv, H_kv, H))
    lens, at = _i32([0, 0]), [0, 0]
    for new in ([64, 40], [1, 0], [85, 57]):
        N = max(new)
        qc, kc, vc = (torch.zeros((R, x.shape[1], N, D), dtype=BF, device=DEV) for x in (q, k, v))
        for b in range(R):
            for c, x in ((qc, q), (kc, k), (vc, v)):
                c[b, :, :new[b]] = x[b, :, at[b]:at[b] + new[b]]
        lengths = _i32(new)
        qr = fa.append_paged(kc, vc, pool.k, pool.v, ptable.to(DEV), lens, lengths=lengths, rotary=rotary, q=qc)
        o, lse = fa.attend_paged(qr, pool.k, pool.v, ptable.to(DEV), lens, lengths=lengths, return_lse=True)
        for b in range(R):
            rq, rk = fa.rotate(q[b:b + 1], k[b:b + 1], 0, rotary)
            assert torch.equal(qr[b, :, :new[b]], rq[0, :, at[b]:at[b] + new[b]])
            top = at[b] + new[b]
            ro, rl, eo, el = attend(rq[0, :, at[b]:top], rk[0, :, :top], v[b, :, :top], [at[b] + i + 1 for i in range(new[b])],
                                    D ** -0.5, BF, N * 4 > 64)
            _near_o(o[b, :, :new[b]], ro, eo, BF, f"prompt {b} from {at[b]}")
            _near(lse[b, :, :new[b]], rl, el, "lse")
            at[b] = top
        lens += lengths
    assert at == sizes and lens.tolist() == sizes
    B = R * n
    table = pool.table([20] * B)
    own = _i32([0] * B)
    ks, vs = (_randn((B, H_kv, 20, D), g, BF) for _ in range(2))
    keys = [[fa.rotate(k[b // n:b // n + 1, :, :sizes[b // n]], None, 0, rotary)[0]] for b in range(B)]
    for i in range(18):
        qi = _randn((B, H, 1, D), g, BF)
        where = (lens.repeat_interleave(n) + i)[:, None]
        qr, kr = fa.rotate(qi, ks[:, :, i:i + 1], where, rotary)
        o, lse = fa.decode_shared(qr[:, :, 0], pool.k, pool.v, ptable.to(DEV), lens, table.to(DEV), own, kr[:, :, 0], vs[:, :, i],
                                  return_lse=True)
        own += 1
        for b in range(B):
            keys[b].append(kr[b])
            if i % 6 == b:
                r = b // n
                ro, rl, eo, el = attend(qr[b], torch.cat(keys[b], 1), torch.cat([v[r, :, :sizes[r]], vs[b, :, :i + 1]], 1),
                                        [sizes[r] + i + 1], D ** -0.5, BF, False)
                _near_o(o[b][:, None], ro, eo, BF, f"sample {b} token {i}")
                _near(lse[b][:, None], rl, el, "lse")
