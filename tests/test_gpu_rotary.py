"""Rotary positions (custom_flash_attn.rotate) and new tokens into a paged cache (append_paged) against the formula in
64 bits (needs a GPU).

Tolerances count roundings, u = 2^-24: an angle below pi / 4 is taken from its integer with three (its own, the
constant's, the product's), so sine and cosine are off by 3 u pi / 4, 0.5 u where their series end and 2 u in them, below
5 u; u more times the magnitude m.  One product is rounded, then the result: 6 u m (|x_a| + |x_b|) + u m |x_b| + u |y|,
at most 8 u m (|x_a| + |x_b|), and half a step of the output's type."""
import math
import sys

import pytest
import torch

import custom_flash_attn as fa

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _randn(shape, g, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g) * sigma).to(dtype).to(DEV)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def turned(x, positions, rotary, transposed=False):
    """x (B, H, N, D) rotated by positions (B, N) in 64 bits on the CPU, and the bound of a result's error before its
    rounding to the type.  Angles come from whole turns in 2^-64, as integers."""
    x = x.detach().double().cpu()
    r, m = rotary.dim, rotary.magnitude
    turns = [t % 2 ** 64 for t in rotary._turns.tolist()]
    phase = [[[(int(p) * t) % 2 ** 64 / 2.0 ** 64 for t in turns] for p in row] for row in positions.tolist()]
    t = 2 * math.pi * torch.tensor(phase, dtype=torch.float64).view(*positions.shape, r // 2)[:, None]
    if transposed:
        t = -t
    a, b = (slice(0, r, 2), slice(1, r, 2)) if rotary.interleaved else (slice(0, r // 2), slice(r // 2, r))
    y, e = x.clone(), torch.zeros_like(x)
    y[..., a] = m * (x[..., a] * t.cos() - x[..., b] * t.sin())
    y[..., b] = m * (x[..., b] * t.cos() + x[..., a] * t.sin())
    e[..., a] = e[..., b] = 8 * U * m * (x[..., a].abs() + x[..., b].abs())
    return y, e


def _near(got, want, bound, dtype, what):
    got = got.detach().double().cpu()
    room = bound + (bound > 0) * (_half(dtype) * (want.abs() + bound) + (2.0 ** -25 if dtype == HF else 0.0))
    d = (got - want).abs()
    _say(f"  {what}: max off {float(d.max()) if d.numel() else 0:.3e}")
    assert torch.isfinite(got).all() and (d <= room).all(), what


CASES = [  # B, H, H_kv, N, D, rot, interleaved, dtype
    (2, 12, 12, 1, 64, 64, False, BF),
    (3, 5, 2, 17, 64, 64, True, BF),
    (1, 8, 2, 130, 128, 64, False, HF),
    (2, 8, 1, 33, 128, 128, True, HF),
    (2, 3, 3, 40, 96, 48, False, F32),
    (1, 4, 4, 25, 40, 20, False, BF),       # halves of 10
    (1, 4, 2, 25, 40, 20, True, HF),
    (2, 2, 2, 9, 80, 80, False, F32),
    (1, 3, 1, 7, 6, 2, True, F32),
    (2, 1, 1, 5, 13, 10, False, BF),        # an odd head
    (1, 1, 0, 1, 2, 2, False, BF),
    (1, 25, 25, 300, 64, 32, True, BF),
    (40, 7, 3, 3, 72, 72, False, HF),
]


@pytest.mark.parametrize("B,H,H_kv,N,D,rot,interleaved,dtype", CASES)
def test_rotate_matches_64_bits(B, H, H_kv, N, D, rot, interleaved, dtype):
    _say(f"rotate B={B} H={H},{H_kv} N={N} D={D} rot={rot} interleaved={interleaved} {dtype}")
    g = _gen(B * 100 + D + rot)
    rotary = fa.Rotary(rot, interleaved=interleaved, magnitude=1.25 if rot == 64 else 1.0, device=DEV)
    q = _randn((B, N, H, D), g, dtype, 2.0).transpose(1, 2)
    k = _randn((B, H_kv, N, D), g, dtype) if H_kv else None
    at = torch.randint(0, 5000, (B, N), generator=g, dtype=torch.int32)
    got = fa.rotate(q, k, at.to(DEV), rotary)
    for x, y, name in ((q, got, "q"),) if k is None else ((q, got[0], "q"), (k, got[1], "k")):
        assert y.shape == x.shape and y.dtype == dtype
        want, bound = turned(x, at, rotary)
        _near(y, want, bound, dtype, name)
        assert torch.equal(y[..., rot:], x[..., rot:])
    # int64, one row for all sequences, and a first position.
    row = torch.arange(N) + 777
    for form in (row.to(DEV), row[None].to(DEV), row[None].int().to(DEV).expand(B, N), 777):
        y = fa.rotate(q, None, form, rotary)
        want, bound = turned(q, row[None].expand(B, N), rotary)
        _near(y, want, bound, dtype, f"positions {type(form)}")


@pytest.mark.parametrize("interleaved,rot", [(False, 64), (True, 64), (False, 20), (True, 20)])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rotate_strides_alignment_and_in_place(interleaved, rot, offset):
    """Views that begin at any element, into outputs of other layouts, and in place; what lies beside is left alone."""
    g = _gen(7 + rot + offset)
    B, H, N, D = 2, 3, 11, 64
    rotary = fa.Rotary(rot, interleaved=interleaved, device=DEV)
    wide = _randn((B, N, H, D + 16), g, BF)
    q = wide[..., offset:offset + D].transpose(1, 2)
    at = torch.arange(N)[None].expand(B, N)
    want, bound = turned(q, at, rotary)
    out = torch.full((H, N, B, D + 16), 7.0, dtype=BF, device=DEV)
    y = fa.rotate(q, None, 0, rotary, q_out=out[..., offset:offset + D].permute(2, 0, 1, 3))
    assert y.data_ptr() == out.data_ptr() + 2 * offset
    _near(y, want, bound, BF, "other layout")
    assert (out[..., :offset] == 7).all() and (out[..., offset + D:] == 7).all()
    before = wide.clone()
    kept = fa.rotate(q, q, 0, rotary, q_out=torch.empty_like(q), k_out=q)[1]
    assert kept.data_ptr() == q.data_ptr()
    _near(q, want, bound, BF, "in place")
    assert torch.equal(wide[..., :offset], before[..., :offset]) and torch.equal(wide[..., offset + D:], before[..., offset + D:])


def test_rotate_far_and_negative_positions():
    g = _gen(8)
    rotary = fa.Rotary(128, base=500000.0, device=DEV)
    at = torch.tensor([[0, 1, -1, 2 ** 20 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 3, -5]])
    q = _randn((1, 4, 8, 128), g, F32)
    want, bound = turned(q, at, rotary)
    _near(fa.rotate(q, None, at.to(DEV), rotary), want, bound, F32, "int64")
    at = at.clamp(-2 ** 31, 2 ** 31 - 1)
    want, bound = turned(q, at, rotary)
    _near(fa.rotate(q, None, at.int().to(DEV), rotary), want, bound, F32, "int32")
    want, bound = turned(q, torch.arange(8)[None] + 2 ** 40, rotary)
    _near(fa.rotate(q, None, 2 ** 40, rotary), want, bound, F32, "first")


def test_rotate_passes_nan_and_infinities_to_their_pairs_only():
    rotary = fa.Rotary(8, device=DEV)
    q = torch.ones(1, 1, 1, 16, dtype=BF, device=DEV)
    q[..., 2], q[..., 9], q[..., 7] = NAN, float("inf"), float("-inf")
    y = fa.rotate(q, None, 3, rotary)[0, 0, 0]
    assert torch.isnan(y[[2, 6]]).all() and y[9] == float("inf") and torch.isinf(y[[3, 7]]).all()
    assert torch.isfinite(y[[0, 1, 4, 5, 8, 10, 11, 12, 13, 14, 15]]).all()


def test_rotate_empty():
    rotary = fa.Rotary(64, device=DEV)
    for shape in ((0, 4, 5, 64), (2, 0, 5, 64), (2, 4, 0, 64)):
        q = torch.empty(shape, dtype=BF, device=DEV)
        assert fa.rotate(q, None, 0, rotary).shape == shape


@pytest.mark.parametrize("interleaved,rot,dtype", [(False, 64, F32), (True, 32, F32), (False, 20, F32), (True, 64, BF), (False, 64, HF)])
def test_rotate_gradients(interleaved, rot, dtype):
    """Against the transposed rotation, and against differences: the rotation is linear, so the difference quotient at
    any step is the derivative, off by what 2 x (B H N D) outputs are off, each weighted."""
    g = _gen(9 + rot)
    B, H, H_kv, N, D = 2, 4, 2, 9, 64
    rotary = fa.Rotary(rot, interleaved=interleaved, magnitude=1.1, device=DEV)
    q = _randn((B, N, H, D), g, dtype).transpose(1, 2).requires_grad_()
    k = _randn((B, H_kv, N, D), g, dtype).requires_grad_()
    at = torch.arange(N, device=DEV) + 40
    wq, wk = _randn(q.shape, g, dtype), _randn(k.shape, g, dtype)
    y = fa.rotate(q, k, at, rotary)
    dq, dk = torch.autograd.grad(y, (q, k), (wq, wk))
    rows = at.cpu()[None].expand(B, N)
    for got, w, name in ((dq, wq, "dq"), (dk, wk, "dk")):
        want, bound = turned(w, rows, rotary, True)
        _near(got, want, bound, dtype, name)
    if dtype == F32:
        d = _randn(q.shape, g, dtype)
        with torch.no_grad():
            up, down = (fa.rotate(q + s * d, None, at, rotary).double() for s in (0.5, -0.5))
        want = ((up - down) * wq.double()).sum()
        # Outputs of |x| up to 6.1 (and x itself rounded once): 20 u m (|x_a| + |x_b|) each, twice.
        room = 2 * 20 * U * 1.1 * 13 * float(wq.abs().double().sum()) + 9 * U * float((dq.double().abs() * d.double().abs()).sum())
        got = (dq.double() * d.double()).sum()
        _say(f"  differences: {float(got):.6f} {float(want):.6f} room {room:.2e}")
        assert abs(float(got - want)) <= room
    # One of the two alone, an expanded gradient, the second derivative.
    only, = torch.autograd.grad(fa.rotate(q, k, at, rotary)[1], (k,), (wk,))
    assert torch.equal(only, dk)
    ones, = torch.autograd.grad(fa.rotate(q, None, at, rotary).sum(), (q,))
    want, bound = turned(torch.ones_like(q), rows, rotary, True)
    _near(ones, want, bound, dtype, "of a sum")
    w = wq.clone().requires_grad_()
    first, = torch.autograd.grad(fa.rotate(q, None, at, rotary), (q,), (w,), create_graph=True)
    again, = torch.autograd.grad(first, (w,), (wk.repeat_interleave(2, 1),))
    want, bound = turned(wk.repeat_interleave(2, 1), rows, rotary)
    _near(again, want, bound, dtype, "second")


def test_rotate_backward_after_the_forward_and_into_leaves():
    g = _gen(11)
    rotary = fa.Rotary(64, device=DEV)
    q = _randn((1, 2, 5, 64), g, F32).requires_grad_()
    (fa.rotate(q, None, 3, rotary) ** 2).sum().backward()
    # The rotation keeps lengths: d|y|^2 = 2 x, off by 2 (8 + 8) u (|x_a| + |x_b|) and the products' roundings.
    assert (q.grad - 2 * q).abs().max() <= 40 * U * 4 * float(q.detach().abs().max())
    with torch.no_grad():
        assert not fa.rotate(q, None, 3, rotary).requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        fa.rotate(q, None, 3, rotary, q_out=torch.empty_like(q))
    at = torch.arange(5, device=DEV)
    y = fa.rotate(q, None, at, rotary)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_rotate_forward_mode_and_function_transforms():
    g = _gen(12)
    rotary = fa.Rotary(64, device=DEV)
    q, t = _randn((1, 2, 5, 64), g, F32), _randn((1, 2, 5, 64), g, F32)
    with torch.autograd.forward_ad.dual_level():
        y = fa.rotate(torch.autograd.forward_ad.make_dual(q, t), None, 2, rotary)
        tangent = torch.autograd.forward_ad.unpack_dual(y).tangent
    want = fa.rotate(t, None, 2, rotary)
    assert torch.equal(tangent, want)
    grad = torch.func.grad(lambda x: (fa.rotate(x, None, 2, rotary) * t).sum())(q)
    x = q.clone().requires_grad_()
    assert torch.equal(grad, torch.autograd.grad((fa.rotate(x, None, 2, rotary) * t).sum(), x)[0])


def test_rotate_in_a_graph_and_on_another_stream():
    g = _gen(13)
    rotary = fa.Rotary(64, device=DEV)
    q, at = _randn((2, 4, 1, 64), g, BF), torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.rotate(q, None, at, rotary)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = fa.rotate(q, None, at, rotary)
            at.add_(1)
    torch.cuda.current_stream().wait_stream(side)
    at.zero_()
    for i in range(4):
        q.copy_(_randn(q.shape, g, BF))
        graph.replay()
        assert torch.equal(y, fa.rotate(q, None, i, rotary))


class Cache:
    """A pool of NaN with each sequence's pages in random order."""

    def __init__(self, g, rows, H_kv, D, page, dtype, rows_first=False, extra=3):
        need = [max(1, -(-n // page)) for n in rows]
        self.P, self.page = sum(need) + extra, page
        order = torch.randperm(self.P, generator=g).tolist()
        shape = (self.P, page, H_kv, D) if rows_first else (self.P, H_kv, page, D)
        self.k, self.v = (torch.full(shape, NAN, dtype=dtype, device=DEV) for _ in range(2))
        if rows_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        table = torch.full((len(rows), max(need)), 2 ** 31 - 9, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.host, self.table = table, table.to(DEV)


def _bits(t):
    return t.contiguous().view(torch.int16)


@pytest.mark.parametrize("H,H_kv,D,N,page,rot,interleaved,dtype,rows_first,queries", [
    (12, 12, 64, 1, 16, 64, False, BF, False, True),
    (25, 25, 64, 70, 64, 0, False, BF, False, False),
    (8, 2, 128, 33, 128, 128, True, HF, True, True),
    (8, 2, 128, 33, 48, 64, False, HF, True, True),
    (4, 4, 40, 19, 7, 20, False, BF, False, True),
    (16, 1, 96, 300, 1, 96, True, BF, False, False),
    (6, 3, 80, 5, 256, 40, False, HF, False, True),
    (3, 3, 8, 2, 16, 2, True, BF, True, True),
])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_paged(H, H_kv, D, N, page, rot, interleaved, dtype, rows_first, queries, ragged):
    _say(f"append H={H},{H_kv} D={D} N={N} page={page} rot={rot} {dtype} ragged={ragged}")
    g = _gen(D + N + page)
    held = [0, 1, page - 1, page, 3 * page + 2]
    new = [N, 0, N // 2, 1, max(0, N - 1)] if ragged else [N] * 5
    c = Cache(g, [h + n for h, n in zip(held, new)], H_kv, D, page, dtype, rows_first)
    k, v = (_randn((5, N, H_kv, D), g, dtype).transpose(1, 2) for _ in range(2))
    q = _randn((5, H, N, D), g, dtype) if queries else None
    rotary = fa.Rotary(rot, interleaved=interleaved, device=DEV) if rot else None
    lens = torch.tensor(held, dtype=torch.int32, device=DEV)
    lengths = torch.tensor(new, dtype=torch.int32, device=DEV) if ragged else None
    for positions in (None, torch.tensor([5, 0, 9, 100000, 7], dtype=torch.int32, device=DEV)) if rot else (None,):
        at = torch.arange(N)[None] + (lens if positions is None else positions).cpu()[:, None]
        k0, v0 = c.k.clone(), c.v.clone()
        got = fa.append_paged(k, v, c.k, c.v, c.table, lens, lengths=lengths, rotary=rotary, positions=positions, q=q)
        for b, (h, n) in enumerate(zip(held, new)):
            for x, pool, before in ((k, c.k, k0), (v, c.v, v0)):
                rows = [(int(c.host[b, j // page]), j % page) for j in range(h, h + n)]
                if rows:
                    pid, off = (torch.tensor(z, device=DEV) for z in zip(*rows))
                    wrote = pool[pid, :, off].transpose(0, 1)[None]
                    if x is k and rot:
                        want, bound = turned(x[b:b + 1, :, :n], at[b:b + 1, :n], rotary)
                        _near(wrote, want, bound, dtype, f"k of {b}")
                    else:
                        assert torch.equal(_bits(wrote), _bits(x[b:b + 1, :, :n]))
                    before[pid, :, off] = pool[pid, :, off]
            if queries:
                want, bound = turned(q[b:b + 1, :, :n], at[b:b + 1, :n], rotary)
                _near(got[b:b + 1, :, :n], want, bound, dtype, f"q of {b}")
                assert (got[b, :, n:] == 0).all()
        assert torch.equal(_bits(c.k), _bits(k0)) and torch.equal(_bits(c.v), _bits(v0))   # no other row
        if not queries:
            assert got is None
    if queries:   # in place, rows past a text's left alone
        mine = q.clone()
        assert fa.append_paged(k, v, c.k, c.v, c.table, lens, lengths=lengths, rotary=rotary, positions=positions, q=mine,
                               q_out=mine) is mine
        for b, n in enumerate(new):
            assert torch.equal(mine[b, :, :n], got[b, :, :n]) and torch.equal(mine[b, :, n:], q[b, :, n:])


def test_append_paged_bad_lengths_and_pages():
    g = _gen(21)
    H, H_kv, D, N, page = 4, 2, 64, 6, 16
    c = Cache(g, [64] * 6, H_kv, D, page, BF)
    table = c.table.clone()
    table[0, 1] = -1         # rows 12..17, of which 16 and 17 have no page
    table[1, 1] = c.P        # rows 20..25: past the pool
    lens = torch.tensor([12, 20, -3, 60, 12, 14], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([6, 6, 6, 5, -1, 7], dtype=torch.int32, device=DEV)
    k, v, q = _randn((6, H_kv, N, D), g, BF), _randn((6, H_kv, N, D), g, BF), _randn((6, H, N, D), g, BF)
    k0 = c.k.clone()
    rotary = fa.Rotary(64, device=DEV)
    got = fa.append_paged(k, v, c.k, c.v, table, lens, lengths=lengths, rotary=rotary, q=q)
    pid = int(c.host[0, 0])
    assert torch.equal(c.v[pid, :, 12:], v[0, :, :4])
    k0[pid, :, 12:] = c.k[pid, :, 12:]
    assert torch.equal(_bits(c.k), _bits(k0))
    assert torch.isfinite(got[:2]).all() and torch.isnan(got[2:]).all()
    # Every page bad: nothing written, nothing read past the table.
    k0, v0 = c.k.clone(), c.v.clone()
    fa.append_paged(k, v, c.k, c.v, torch.full_like(table, 2 ** 31 - 1), lens.clamp(0, 50))
    assert torch.equal(_bits(c.k), _bits(k0)) and torch.equal(_bits(c.v), _bits(v0))


def test_append_paged_large_offsets():
    """A pool of more than 2^31 elements: rows past 4 GiB."""
    P, H_kv, page, D = 40, 8, 65536, 128
    pool = torch.zeros((2, P, H_kv, page, D), dtype=BF, device=DEV)
    table = torch.tensor([[39, 38]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([page - 1], dtype=torch.int32, device=DEV)
    k, v = _randn((1, H_kv, 2, D), _gen(22), BF), _randn((1, H_kv, 2, D), _gen(23), BF)
    fa.append_paged(k, v, pool[0], pool[1], table, lens)
    for x, p in ((k, pool[0]), (v, pool[1])):
        assert torch.equal(p[39, :, page - 1], x[0, :, 0]) and torch.equal(p[38, :, 0], x[0, :, 1])
        assert int(p.view(-1, D).any(-1).sum()) == 2 * H_kv


def test_append_paged_in_a_graph():
    g = _gen(24)
    H_kv, D, page = 4, 64, 16
    c = Cache(g, [64, 64], H_kv, D, page, BF)
    lens = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    rotary = fa.Rotary(64, device=DEV)
    k, v, q = (_randn((2, H_kv, 1, D), g, BF) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.append_paged(k, v, c.k, c.v, c.table, lens, rotary=rotary, q=q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = fa.append_paged(k, v, c.k, c.v, c.table, lens, rotary=rotary, q=q)
            lens.add_(1)
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(torch.tensor([0, 20], dtype=torch.int32))
    for i in range(20):
        for x in (k, v, q):
            x.copy_(_randn(x.shape, g, BF))
        graph.replay()
        at = torch.tensor([[i], [20 + i]], device=DEV)
        kr, qr = fa.rotate(k, q, at, rotary)
        for b, j in ((0, i), (1, 20 + i)):
            pid = int(c.host[b, j // page])
            assert torch.equal(c.k[pid, :, j % page], kr[b, :, 0]) and torch.equal(c.v[pid, :, j % page], v[b, :, 0])
        assert torch.equal(y, qr)
