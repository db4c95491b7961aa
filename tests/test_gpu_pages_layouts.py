"""Layouts: inputs whose new results torch would lay out otherwise, and parts in their workspaces (needs a
GPU)."""
import pytest
import torch

import custom_flash_attn as fa

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _randn(*shape, dtype=F32):
    return torch.randn(shape, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape,strides", [
    ((1, 1, 3, 8), (0, 0, 1, 1)),          # a window that slides over a row by one
    ((1, 2, 5, 64), (0, 7, 1, 1)),
    ((2, 3, 4, 16), (1, 1, 1, 1)),
    ((2, 3, 4, 16), (0, 0, 8, 1)),
    ((2, 3, 4, 16), (0, 0, 0, 1)),         # one row for all
])
def test_rotation_of_rows_over_one_another(dtype, shape, strides):
    """Inputs whose rows share elements, and gradients that do."""
    rotary = fa.Rotary(shape[3], device=DEV)
    base = _randn(400, dtype=dtype)
    x = base.as_strided(shape, strides)
    want = fa.rotate(x.contiguous(), None, 5, rotary)
    assert torch.equal(fa.rotate(x, None, 5, rotary), want)
    a, b = fa.rotate(x, x, 5, rotary)
    assert torch.equal(a, want) and torch.equal(b, want)
    b = torch.empty_like(want)
    a, b = fa.rotate(x, x, 5, rotary, k_out=b)
    assert torch.equal(a, want) and torch.equal(b, want)
    z = _randn(*shape, dtype=dtype).requires_grad_()
    g, = torch.autograd.grad(fa.rotate(z, None, 5, rotary), z, x)
    assert torch.equal(g, torch.autograd.grad(fa.rotate(z, None, 5, rotary), z, x.contiguous())[0])


@pytest.mark.parametrize("strides", [(1, 0, 0, 1), (1, 0, 1, 1), (0, 0, 64, 1)])
def test_one_token_expanded_over_heads(strides):
    """A token's query row for all heads, where dimensions of one element have strides of their own."""
    H, H_kv, D = 4, 2, 64
    k_pages, v_pages = (torch.zeros(2, H_kv, 16, D, dtype=BF, device=DEV) for _ in range(2))
    table, lens = torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    k, v = _randn(1, H_kv, 1, D, dtype=BF), _randn(1, H_kv, 1, D, dtype=BF)
    q = _randn(D, dtype=BF).as_strided((1, H, 1, D), strides)
    rotary = fa.Rotary(64, device=DEV)
    got = fa.append_paged(k, v, k_pages, v_pages, table, lens, rotary=rotary, q=q)
    assert torch.equal(got, fa.append_paged(k, v, k_pages, v_pages, table, lens, rotary=rotary, q=q.contiguous()))
    assert torch.equal(fa.attend_paged(q, k_pages, v_pages, table, lens),
                       fa.attend_paged(q.contiguous(), k_pages, v_pages, table, lens))
    assert torch.equal(fa.rotate(q, None, 3, rotary), fa.rotate(q.contiguous(), None, 3, rotary))


@pytest.mark.parametrize("H,H_kv,D,R,n", [(3, 3, 64, 1, 4), (6, 2, 128, 2, 5), (40, 1, 64, 1, 3), (5, 5, 72, 1, 70)])
def test_workspaces_of_just_the_size(H, H_kv, D, R, n):
    """Parts of few rows, of a tile and of several lie in the bytes that are asked for, and give what a larger workspace
    gives."""
    page, M_prefix, M, B = 16, 300, 40, R * n
    g = torch.Generator().manual_seed(H + D)
    k_pages, v_pages = (torch.randn(R * M_prefix + B * M, H_kv, page, D, generator=g).to(BF).to(DEV) for _ in range(2))
    order = torch.randperm(R * M_prefix + B * M, generator=g).to(torch.int32).to(DEV)
    prefix, table = order[:R * M_prefix].view(R, M_prefix), order[R * M_prefix:].view(B, M)
    plens = torch.full((R,), M_prefix * page - 3, dtype=torch.int32, device=DEV)
    lens = torch.arange(B, dtype=torch.int32, device=DEV) * 9
    C = fa._C

    def check(call, nbytes):
        assert nbytes > 0
        want = call(torch.empty(2 * nbytes, dtype=torch.uint8, device=DEV))
        room = torch.full((nbytes + 256,), 255, dtype=torch.uint8, device=DEV)
        got = call(room[:nbytes])
        assert (room[nbytes:] == 255).all()
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, want))

    q = torch.randn(B, H, D, generator=g).to(BF).to(DEV)
    check(lambda ws: fa.decode_shared(q, k_pages, v_pages, prefix, plens, table, lens, return_lse=True, workspace=ws),
          C.decode_shared_workspace(R, B, H, H_kv, page, M_prefix, M, D))
    for N in (1, 2, n):
        x = torch.randn(R, H, N, D, generator=g).to(BF).to(DEV)
        check(lambda ws: fa.attend_paged(x, k_pages, v_pages, prefix, plens - N, return_lse=True, workspace=ws),
              C.attend_workspace(R, H, H_kv, N, page, M_prefix, D))
