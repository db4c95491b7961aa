"""Scores of any finite size in the attention of several rows over a paged cache (custom_flash_attn.attend_paged,
decode_shared), whose kernels for many and for few rows hold offsets differently (needs a GPU).

A score is one product q k of few bits, exact in float32, so that the softmax is known: equal keys give the mean of the
values, a key whose score is above the others' by at least 2^10 gives its value.  u = 2^-24, half =
torch.finfo(type).eps / 2.  Tolerances:
  * the mean of L values: equal weights, rounded alike, cancel in the division; sums of L terms are off by (L + 16) u, the
    output's rounding by half;
  * the one value: its weight over itself, so the value, which is of the output's type;
  * the log-sum-exp x + ln L: two roundings of x in the offset, one in its product with the scale and one in the sum (4 u
    |x|); the logarithm, up to 40, by 4 u of it, its argument by (L + 16) u."""
import math

import pytest
import torch

import custom_flash_attn as fa

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
BF, HF = torch.bfloat16, torch.float16
D, PAGE = 64, 16
# (exponent of q, exponent of k, scale): scores of 2^16 to 2^119 on both sides of where float32 holds whole numbers only.
SIZES = [(10, 8, 0.3), (10, 10, 0.3), (12, 11, 0.3), (13, 12, 0.3), (14, 13, 0.3), (15, 13, 0.125), (15, 14, 0.3), (15, 15, 0.3),
         (14, 14, 0.3 * 2.0 ** 5), (15, 15, 0.3 * 2.0 ** 12), (15, 15, 0.3 * 2.0 ** 30), (15, 15, 0.3 * 2.0 ** 70),
         (15, 15, 0.3 * 2.0 ** 89)]
MANTISSAS = [1 + n / 64 for n in (0, 3, 7, 10, 17, 21, 24, 29, 33, 38, 42, 47, 51, 55, 60, 63)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _expected(v, lo, top, scale, seen):
    """o and lse of rows that see the first `seen` keys, of raw score lo but for key 17, of raw score top."""
    if lo == top:
        return v[:seen].double().mean(0), _f32(scale) * lo + math.log(seen)
    return v[17].double(), _f32(scale) * top


def _check(o, lse, v, lo, top, scale, seen, half, what):
    want, x = _expected(v, lo, top, scale, seen)
    if lo == top:
        room = ((seen + 16) * U + 1.01 * half) * v[:seen].double().abs().mean(0)
        assert ((o.double() - want).abs() <= room).all(), (what, o.tolist()[:4], want.tolist()[:4])
    else:
        assert torch.equal(o.double(), want), (what, o.tolist()[:4], want.tolist()[:4])
    assert abs(float(lse) - x) <= 4 * U * abs(x) + (seen + 16 + 160) * U, (what, float(lse), x)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("N,L", [(2, 40), (65, 40), (129, 70), (129, 6000)])
def test_attend_paged_scores_of_any_size(dtype, sign, alone, N, L):
    """One sequence a mantissa of q; all rows of a tile have the same scores, and the last tile of 65 or 129 rows one row.
    (6000 rows before the tokens: keys divided over workgroups.)"""
    g = torch.Generator().manual_seed(N + L)
    B, M, half = len(MANTISSAS), -(-(L + N) // PAGE), torch.finfo(dtype).eps / 2
    v = torch.randn((B, L + N, D), generator=g).to(dtype).to(DEV)
    table = torch.randperm(B * M, generator=g).to(torch.int32).to(DEV).view(B, M)
    k_pages, v_pages = (torch.zeros(B * M, 1, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
    lens = _i32([L] * B)
    for eq, ek, scale in SIZES:
        k = torch.zeros(B, 1, L + N, D, dtype=dtype, device=DEV)
        k[..., 0] = sign * 2.0 ** ek
        if alone:
            k[:, :, 17, 0] = sign * 2.0 ** ek * (1 + sign * 2.0 ** -5)
        fa.append_paged(k, v[:, None], k_pages, v_pages, table, _i32([0] * B))
        q = torch.zeros(B, 1, N, D, dtype=dtype, device=DEV)
        q[..., 0] = torch.tensor(MANTISSAS, device=DEV).view(B, 1, 1) * 2.0 ** eq
        o, lse = fa.attend_paged(q, k_pages, v_pages, table, lens, softmax_scale=scale, return_lse=True)
        plain = fa.attend_paged(q, k_pages, v_pages, table, lens, softmax_scale=scale)
        assert torch.equal(o, plain)
        for b, a in enumerate(MANTISSAS):
            lo = sign * a * 2.0 ** (eq + ek)
            for i in (0, N - 1):
                _check(o[b, 0, i], lse[b, 0, i], v[b], lo, lo * (1 + sign * 2.0 ** -5) if alone else lo, scale, L + i + 1, half,
                       (eq, ek, scale, a, i))


@pytest.mark.parametrize("n", [3, 70])
def test_attend_paged_and_decode_shared_of_twenty_thousands(n):
    """Queries and keys of 20000 in every dim, scale 1/8, fp16: scores of 3.2e9."""
    g = torch.Generator().manual_seed(n)
    L, half = 100, torch.finfo(HF).eps / 2
    M = -(-(L + n) // PAGE)
    v = torch.randn((L + n, D), generator=g).to(HF).to(DEV)
    k = torch.full((1, 1, L + n, D), 20000.0, dtype=HF, device=DEV)
    k_pages, v_pages = (torch.zeros(M, 1, PAGE, D, dtype=HF, device=DEV) for _ in range(2))
    table = torch.arange(M, dtype=torch.int32, device=DEV)[None]
    fa.append_paged(k, v[None, None], k_pages, v_pages, table, _i32([0]))
    raw = 20000.0 ** 2 * D
    o, lse = fa.attend_paged(k[:, :, :n].contiguous(), k_pages, v_pages, table, _i32([L]), return_lse=True)
    for i in (0, n - 1):
        _check(o[0, 0, i], lse[0, 0, i], v, raw, raw, 0.125, L + i + 1, half, i)
    o, lse = fa.decode_shared(k[0, 0, :n, None].contiguous(), k_pages, v_pages, table, _i32([L]),
                              torch.zeros(n, 0, dtype=torch.int32, device=DEV), _i32([0] * n), return_lse=True)
    for i in (0, n - 1):
        _check(o[i, 0], lse[i, 0], v, raw, raw, 0.125, L, half, i)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("B,L", [(5, 50), (70, 50), (130, 50), (70, 6000)])
def test_decode_shared_scores_of_any_size(dtype, sign, alone, B, L):
    """One key-value head a mantissa of q, B sequences behind one prefix with two rows of their own."""
    g = torch.Generator().manual_seed(B + L)
    H, half, M = len(MANTISSAS), torch.finfo(dtype).eps / 2, -(-L // PAGE)
    v = torch.randn((H, L, D), generator=g).to(dtype).to(DEV)
    own = torch.randn((B, H, 2, D), generator=g).to(dtype).to(DEV)
    order = torch.randperm(M + B, generator=g).to(torch.int32).to(DEV)
    prefix, table = order[None, :M], order[M:, None]
    k_pages, v_pages = (torch.zeros(M + B, H, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
    for eq, ek, scale in SIZES:
        k = torch.zeros(1, H, L, D, dtype=dtype, device=DEV)
        k[..., 0] = sign * 2.0 ** ek
        if alone:
            k[:, :, 17, 0] = sign * 2.0 ** ek * (1 + sign * 2.0 ** -5)
        fa.append_paged(k, v[None], k_pages, v_pages, prefix, _i32([0]))
        fa.append_paged(k[:, :, :2].expand(B, H, 2, D), own, k_pages, v_pages, table, _i32([0] * B))
        q = torch.zeros(B, H, D, dtype=dtype, device=DEV)
        q[..., 0] = torch.tensor(MANTISSAS, device=DEV) * 2.0 ** eq
        o, lse = fa.decode_shared(q, k_pages, v_pages, prefix, _i32([L]), table, _i32([2] * B), softmax_scale=scale, return_lse=True)
        for h, a in enumerate(MANTISSAS):
            lo = sign * a * 2.0 ** (eq + ek)
            for b in (0, B - 1):
                _check(o[b, h], lse[b, h], torch.cat([v[h], own[b, h]]), lo, lo * (1 + sign * 2.0 ** -5) if alone else lo, scale,
                       L + 2, half, (eq, ek, scale, a, b))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N", [2, 100])
def test_attend_paged_differences_beside_large_scores(dtype, N):
    """Scores of 2^26, where float32 holds multiples of 8, and one 16 above: the weights are of the differences."""
    g = torch.Generator().manual_seed(N)
    L, M, half = 300, -(-(300 + N) // PAGE), torch.finfo(dtype).eps / 2
    v = torch.randn((1, 1, L + N, D), generator=g).to(dtype).to(DEV)
    k = torch.zeros(1, 1, L + N, D, dtype=dtype, device=DEV)
    k[..., 0], k[0, 0, 128, 1] = 2.0 ** 11, 16
    k_pages, v_pages = (torch.zeros(M, 1, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
    table = torch.arange(M, dtype=torch.int32, device=DEV)[None]
    fa.append_paged(k, v, k_pages, v_pages, table, _i32([0]))
    q = torch.zeros(1, 1, N, D, dtype=dtype, device=DEV)
    q[..., 0], q[..., 1] = 2.0 ** 15, 1
    o = fa.attend_paged(q, k_pages, v_pages, table, _i32([L]), softmax_scale=0.3)
    # (Differences of 16 by the scale: 2 u 4.8; the weights' bits: 2 half, or 2^-16 in two parts.)
    w = 2 * half if N > 64 else 2.0 ** -16
    for i in (0, N - 1):
        p = torch.softmax(k[0, 0, :L + i + 1, 1].double() * 0.3, 0)
        vv = v[0, 0, :L + i + 1].double()
        room = ((L + N + 32) * U + 10 * U + w + 1.01 * half) * (p @ vv.abs())
        assert ((o[0, 0, i].double() - p @ vv).abs() <= room).all(), i


@pytest.mark.parametrize("dtype", [BF, HF])
def test_attend_paged_no_score_but_the_lowest(dtype):
    """Keys of score -inf before keys whose scaled scores are below float32's range: those share the weight."""
    N, L, half = 128, 96, torch.finfo(dtype).eps / 2   # (a whole tile of rows)
    M = -(-(L + N) // PAGE)
    g = torch.Generator().manual_seed(3)
    v = torch.randn((1, 1, L + N, D), generator=g).to(dtype).to(DEV)
    k = torch.zeros(1, 1, L + N, D, dtype=dtype, device=DEV)
    k[..., 0] = -2.0 ** 15
    k[:, :, :64, 0] = -math.inf
    k_pages, v_pages = (torch.zeros(M, 1, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
    table = torch.arange(M, dtype=torch.int32, device=DEV)[None]
    fa.append_paged(k, v, k_pages, v_pages, table, _i32([0]))
    q = torch.full((1, 1, N, D), 0.0, dtype=dtype, device=DEV)
    q[..., 0] = 2.0 ** 14
    # -2^29 2^98.6 log2 e: past -2^128.
    o = fa.attend_paged(q, k_pages, v_pages, table, _i32([L]), softmax_scale=1.5 * 2.0 ** 98)
    for i in (0, N - 1):
        vv = v[0, 0, 64:L + i + 1].double()
        assert ((o[0, 0, i].double() - vv.mean(0)).abs() <= ((L + N + 16) * U + 1.01 * half) * vv.abs().mean(0)).all(), i
