"""What the operators around a paged cache tell autograd: which results are part of a graph, and that tensors of the
caller's were written (needs a GPU)."""
import pytest
import torch

import custom_flash_attn as fa

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _randn(*shape, dtype=F32):
    return torch.randn(shape, device=DEV).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(B, H_kv, D=64, page=16, M=4):
    k_pages, v_pages = (torch.zeros(B * M, H_kv, page, D, dtype=BF, device=DEV) for _ in range(2))
    return k_pages, v_pages, torch.arange(B * M, dtype=torch.int32, device=DEV).view(B, M)


def test_in_place_rotation_of_a_saved_tensor_is_noticed():
    rotary = fa.Rotary(64, device=DEV)
    q, k, w = _randn(1, 2, 5, 64), _randn(1, 2, 5, 64), _randn(1, 2, 5, 64).requires_grad_()
    for x, given in ((q, dict(q_out=q)), (k, dict(q_out=torch.empty_like(q), k_out=k))):
        y = w * x
        fa.rotate(q, k, 0, rotary, **given)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    y = w * q                       # (nothing of q is written here)
    fa.rotate(q, k, 0, rotary, k_out=k)
    fa.rotate(q, k, 0, rotary)
    y.sum().backward()
    assert torch.equal(w.grad, q)


def test_what_the_paged_operators_write_is_noticed():
    B, H, H_kv, N, D = 2, 4, 2, 3, 64
    k_pages, v_pages, table = _cache(B, H_kv)
    q, k, v = _randn(B, H, N, D, dtype=BF), _randn(B, H_kv, N, D, dtype=BF), _randn(B, H_kv, N, D, dtype=BF)
    lens, out, vec = _i32([5, 7]), torch.zeros(B, H, N, D, dtype=BF, device=DEV), torch.zeros(B, H, D, dtype=BF, device=DEV)
    prefix, plens = table[:1, :1].contiguous(), _i32([5])
    rotary = fa.Rotary(64, device=DEV)
    calls = [
        (lambda: fa.append_paged(k, v, k_pages, v_pages, table, lens, rotary=rotary, q=q, q_out=q), [k_pages, v_pages, q]),
        (lambda: fa.append_paged(k, v, k_pages, v_pages, table, lens), [k_pages, v_pages]),
        (lambda: fa.attend_paged(q, k_pages, v_pages, table, lens, out=out), [out]),
        (lambda: fa.attend_paged(q, k_pages, v_pages, table, lens), []),
        (lambda: fa.decode_shared(q[:, :, 0], k_pages, v_pages, prefix, plens, table, lens, k[:, :, 0], v[:, :, 0], out=vec),
         [k_pages, v_pages, vec]),
        (lambda: fa.decode_shared(q[:, :, 0], k_pages, v_pages, prefix, plens, table, lens, out=vec), [vec]),
        (lambda: fa.decode_shared(q[:, :, 0], k_pages, v_pages, prefix, plens, table, lens), []),
    ]
    everything = [q, k, v, k_pages, v_pages, table, lens, out, vec, prefix, plens]
    for n, (call, written) in enumerate(calls):
        before = [t._version for t in everything]
        call()
        for i, (t, was) in enumerate(zip(everything, before)):
            assert (t._version > was) == any(t is x for x in written), (n, i)
    with torch.inference_mode():
        pools = [x.clone() for x in (k_pages, v_pages)]
        fa.append_paged(k, v, *pools, table, lens)
    fa.append_paged(k, v, *pools, table, lens)   # inference tensors have no versions
    torch.cuda.synchronize()


def test_outputs_that_require_a_gradient_are_refused():
    B, H, N, D = 2, 2, 3, 64
    k_pages, v_pages, table = _cache(B, H)
    x, lens, rotary = _randn(B, H, N, D, dtype=BF), _i32([5, 7]), fa.Rotary(64, device=DEV)
    out = torch.zeros_like(x).requires_grad_()
    vec = torch.zeros(B, H, D, dtype=BF, device=DEV).requires_grad_()
    pool = k_pages.clone().requires_grad_()
    calls = [lambda: fa.rotate(x, None, 0, rotary, q_out=out),
             lambda: fa.rotate(x, x, 0, rotary, k_out=out),
             lambda: fa.append_paged(x, x, k_pages, v_pages, table, lens, rotary=rotary, q=x, q_out=out),
             lambda: fa.append_paged(x, x, pool, v_pages, table, lens),
             lambda: fa.append_paged(x, x, k_pages, pool, table, lens),
             lambda: fa.attend_paged(x, k_pages, v_pages, table, lens, out=out),
             lambda: fa.decode_shared(x[:, :, 0], k_pages, v_pages, table[:1], lens[:1], table, lens, out=vec),
             lambda: fa.decode_shared(x[:, :, 0], pool, v_pages, table[:1], lens[:1], table, lens, x[:, :, 0], x[:, :, 0])]
    for call in calls:
        with pytest.raises(RuntimeError, match="not differentiable"):
            call()
        with torch.no_grad():
            call()
    fa.attend_paged(x, pool, v_pages, table, lens)   # (only read)
    torch.cuda.synchronize()


def test_tangents_of_one_of_two_inputs():
    """Forward mode where queries or keys alone have a tangent, by themselves, in a transform, and over a gradient."""
    rotary, fad = fa.Rotary(64, device=DEV), torch.autograd.forward_ad
    q, k, t = _randn(1, 4, 5, 64), _randn(1, 2, 5, 64), _randn(1, 4, 5, 64)
    rq, rk, rt = (fa.rotate(x, None, 3, rotary) for x in (q, k, t))
    for which in range(2):
        with fad.dual_level():
            pair = [q, k]
            pair[which] = fad.make_dual(pair[which], t[:, :pair[which].shape[1]])
            outs = [fad.unpack_dual(y) for y in fa.rotate(*pair, 3, rotary)]
        assert torch.equal(outs[0].primal, rq) and torch.equal(outs[1].primal, rk)
        assert torch.equal(outs[which].tangent, rt[:, :pair[which].shape[1]])
        other = outs[1 - which].tangent
        assert other is None or (other == 0).all()
    (a, b), (da, db) = torch.func.jvp(lambda x: fa.rotate(x, k, 3, rotary), (q,), (t,))
    assert torch.equal(a, rq) and torch.equal(b, rk) and torch.equal(da, rt) and (db == 0).all()
    # The rotation keeps lengths: the gradient of its half square is x, the derivative of that t.  Two rotations of |x| up to
    # 6, each off by 20 u (|x_a| + |x_b|).
    _, h = torch.func.jvp(torch.func.grad(lambda x: (fa.rotate(x, k, 3, rotary)[0] ** 2).sum() / 2), (q,), (t,))
    assert (h - t).abs().max() <= 2 * 20 * 2.0 ** -24 * 2 * float(t.abs().max())


def test_rotation_of_an_input_without_gradient_is_outside_the_graph():
    rotary = fa.Rotary(64, device=DEV)
    q, k = _randn(1, 4, 5, 64), _randn(1, 2, 5, 64)
    for first, second in ((True, False), (False, True), (True, True), (False, False)):
        x, y = q.clone().requires_grad_(first), k.clone().requires_grad_(second)
        a, b = fa.rotate(x, y, 3, rotary)
        assert (a.requires_grad, b.requires_grad) == (first, second)
        want = fa.rotate(q, k, 3, rotary)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
        for z, out in ((x, a), (y, b)):
            if z.requires_grad:
                g, = torch.autograd.grad(out.sum(), z, retain_graph=True)
                assert torch.equal(g, torch.autograd.grad(fa.rotate(z, None, 3, rotary).sum(), z)[0])
    # A tangent of one input only, beside a gradient of the other.
    with torch.autograd.forward_ad.dual_level():
        x = q.clone().requires_grad_()
        a, b = fa.rotate(x, torch.autograd.forward_ad.make_dual(k, k), 3, rotary)
        assert torch.equal(torch.autograd.forward_ad.unpack_dual(b).tangent, want[1])
        g, = torch.autograd.grad(a.sum(), x)
    assert torch.equal(g, torch.autograd.grad(fa.rotate(x, None, 3, rotary).sum(), x)[0])
