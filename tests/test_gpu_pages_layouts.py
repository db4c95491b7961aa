"""Layouts that the operators around a paged cache take and whose new results torch would lay out otherwise (needs a
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
