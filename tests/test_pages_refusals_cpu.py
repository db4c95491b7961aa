"""More refusals of the operators around a paged cache, on the CPU: with tensors that say they are on a device, and nothing
launched."""
import ctypes

import pytest
import torch

import custom_flash_attn as fa
import test_pages_cpu as boundary
from custom_flash_attn import pages

BF, I32 = torch.bfloat16, torch.int32


class _Dev(torch.Tensor):
    """A CPU tensor that calls itself a device's."""

    is_cuda = True

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        with torch._C.DisableTorchFunctionSubclass():
            return func(*args, **(kwargs or {}))


def _dev(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Dev)


@pytest.fixture
def launches(monkeypatch):
    """Calls that reach the launch."""
    calls = []
    monkeypatch.setattr(pages, "_launch_on", lambda index, fn, *args: calls.append(args))
    monkeypatch.setattr(pages, "_workspace", lambda given, index, nbytes: None)
    return calls


def _grad(t):
    return t.detach().requires_grad_().as_subclass(_Dev)


def test_written_tensors_that_require_a_gradient(launches):
    x, vec, pool, table, lens = _dev(2, 2, 3, 64), _dev(2, 2, 64), _dev(8, 2, 16, 64), _dev(2, 4, dtype=I32), _dev(2, dtype=I32)
    rotary = fa.Rotary(64, device="cpu")
    calls = [lambda: fa.rotate(x, None, 0, rotary, q_out=_grad(x)),
             lambda: fa.rotate(x, x, 0, rotary, k_out=_grad(x)),
             lambda: fa.append_paged(x, x, pool, pool, table, lens, rotary=rotary, q=x, q_out=_grad(x)),
             lambda: fa.append_paged(x, x, _grad(pool), pool, table, lens),
             lambda: fa.append_paged(x, x, pool, _grad(pool), table, lens),
             lambda: fa.attend_paged(x, pool, pool, table, lens, out=_grad(x)),
             lambda: fa.decode_shared(vec, pool, pool, table, lens, table, lens, out=_grad(vec)),
             lambda: fa.decode_shared(vec, pool, _grad(pool), table, lens, table, lens, vec, vec)]
    for call in calls:
        with pytest.raises(RuntimeError, match="not differentiable"):
            call()
    assert not launches
    with torch.no_grad():
        for call in calls:
            call()
    assert len(launches) == len(calls)
    fa.attend_paged(x, _grad(pool), pool, table, lens)                          # (only read)
    fa.decode_shared(vec, _grad(pool), pool, table, lens, table, lens)
    assert len(launches) == len(calls) + 2


def test_workspaces_hold_the_rows_that_there_are():
    """A part keeps D sums, an offset and two sums of weights of each of its rows, in whole lines of 128 bytes, all of them in
    256 bytes."""
    C = pages._C

    def at_most(jobs, parts, rows, D):
        return jobs * parts * (rows * (D + 3) + 31) // 32 * 128 + 256

    # (groups, sequences, query heads, key-value heads, page, prefix pages, pages, D): own parts of one row, of four, of 40 heads
    # in two tiles; jobs enough for one part each.
    assert C.decode_shared_workspace(1, 512, 32, 32, 16, 64, 8, 128) <= at_most(32 * 4, 2, 128, 128) + at_most(512 * 32, 1, 1, 128)
    assert C.decode_shared_workspace(8, 512, 32, 8, 16, 64, 8, 128) <= at_most(8 * 8 * 2, 2, 128, 128) + at_most(512 * 8, 1, 4, 128)
    assert C.decode_shared_workspace(1, 600, 40, 1, 16, 8, 8, 64) <= at_most(188, 1, 128, 64) + at_most(600 * 2, 1, 32, 64)
    assert C.decode_shared_workspace(2, 6, 12, 12, 16, 2048, 8, 64) <= at_most(24, 21, 3, 64) + at_most(72, 1, 1, 64)
    # One token of one query head a key-value head behind a long cache.
    assert C.attend_workspace(1, 12, 12, 1, 16, 2048, 64) <= at_most(12, 32, 1, 64)
    assert C.attend_workspace(1, 12, 12, 70, 16, 2048, 64) <= at_most(12, 32, 70, 64)


@pytest.mark.parametrize("kw,match", [
    (dict(base=1e-320), "float64's range"),
    (dict(scaling="base", factor=10.0, base=1e308), "float64's range"),      # a base past it: all frequencies 0 but the first
    (dict(scaling="base", factor=1e-200, base=1e-200), "float64's range"),   # a base of 0
    (dict(scaling="base", factor=1e300, dim=4), "float64's range"),
    (dict(scaling="linear", factor=1e-320), "float64's range"),
    (dict(scaling="bands", factor=1e-320, trained_length=10), "float64's range"),
    (dict(scaling="bands", factor=2.0, trained_length=float("nan")), "trained_length"),
])
def test_rotary_refuses_numbers_past_its_range(kw, match):
    kw = dict(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.Rotary(kw.pop("dim", 64), device="cpu", **kw)


def test_rotary_of_unusual_bases():
    assert fa.Rotary(2, 1e-300, device="cpu").frequencies == (1.0,)
    assert fa.Rotary(2, scaling="base", factor=1e300, device="cpu").frequencies == (1.0,)
    assert fa.Rotary(4, 1e300, device="cpu").frequencies == (1.0, 1e-150)
    assert fa.Rotary(4, 0.25, device="cpu").frequencies == (1.0, 2.0)


def test_first_positions_of_64_bits(launches):
    x, rotary = _dev(2, 2, 3, 64), fa.Rotary(64, device="cpu")
    for p in (2 ** 63, -2 ** 63 - 1, 10 ** 30):
        with pytest.raises(RuntimeError, match="64 bits"):
            fa.rotate(x, None, p, rotary)
    assert not launches
    for p in (2 ** 63 - 1, -2 ** 63, 0, True):
        fa.rotate(x, None, p, rotary)
    assert len(launches) == 4


def test_scales_whose_binary_logarithm_form_is_infinite():
    """Weights are 2^(scale log2 e (s - m)): a scale of 2.4e38 or more would be infinite in it, and equal scores NaN."""
    lib = ctypes.CDLL(fa.library_path())
    for call in (boundary._attend, boundary._shared):
        assert call(lib, scale=2.4e38) == boundary._code("ERR_SCALE")
        assert call(lib, scale=3.4e38) == boundary._code("ERR_SCALE")
        assert call(lib, scale=2.3e38, q=0) == boundary._code("ERR_NULL_POINTER")
