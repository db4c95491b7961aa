"""CPU-side tests of the serving operators' boundary (include/tfgfa_serving.h): every refusal of the C ABI and of
the Python functions, and the sizes of workspaces.  No kernel is launched: argument checks come before any HIP
call, and every call here fails them or has nothing to do."""
import ctypes
import os
import re
import weakref

import pytest
import torch

import custom_flash_attn as fa
from custom_flash_attn import _C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
P = 0x10000  # a pointer that is never dereferenced
I64 = ctypes.c_int64


def _code(name):
    return int(re.search(rf"#define\s+TFGFA_{name}\s+(-?\d+)", open(os.path.join(INCLUDE, "tfgfa.h")).read()).group(1))


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(fa.library_path())


def test_library_exports_the_serving_entry_points(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INCLUDE, "tfgfa_serving.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(tfserve_\w+)\s*\(", text)))
    assert names == ["tfserve_decode_paged", "tfserve_decode_paged_workspace", "tfserve_evict", "tfserve_key_weights",
                     "tfserve_key_weights_workspace", "tfserve_penalize"]
    assert all(hasattr(lib, n) for n in names) and lib.tfgfa_abi_version() >= 10


def _ptr(x):
    return ctypes.c_void_p(x)


def _strides(*v):
    return (I64 * len(v))(*v)


def _paged(lib, **kw):
    a = dict(q=P, qs=(256, 64, 1), k=P, ks=(4096, 1024, 64, 1), v=P, vs=(4096, 1024, 64, 1), table=P, ts=8, lens=P,
             kn=0, kns=(256, 64, 1), vn=0, vns=(256, 64, 1), o=P, os=(256, 64, 1), lse=0, w=0, ws=(512, 128), B=2,
             H=4, Hkv=4, pages=10, page=16, M=8, D=64, dtype=0, scale=0.125, work=0, bytes=0)
    a.update(kw)
    return lib.tfserve_decode_paged(
        _ptr(a["q"]), _strides(*a["qs"]), _ptr(a["k"]), _strides(*a["ks"]), _ptr(a["v"]), _strides(*a["vs"]),
        _ptr(a["table"]), I64(a["ts"]), _ptr(a["lens"]), _ptr(a["kn"]), _strides(*a["kns"]), _ptr(a["vn"]),
        _strides(*a["vns"]), _ptr(a["o"]), _strides(*a["os"]), _ptr(a["lse"]), _ptr(a["w"]), _strides(*a["ws"]),
        a["B"], a["H"], a["Hkv"], a["pages"], a["page"], a["M"], a["D"], a["dtype"], ctypes.c_float(a["scale"]),
        _ptr(a["work"]), ctypes.c_size_t(a["bytes"]), _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), "ERR_DTYPE"),
    (dict(B=-1), "ERR_BAD_SHAPE"),
    (dict(H=6), "ERR_BAD_SHAPE"),                 # not a multiple of the cache's heads
    (dict(Hkv=0), "ERR_BAD_SHAPE"),
    (dict(page=0), "ERR_BAD_SHAPE"),
    (dict(M=-1), "ERR_BAD_SHAPE"),
    (dict(pages=0), "ERR_BAD_SHAPE"),             # a sequence, but no page
    (dict(D=60), "ERR_HEAD_DIM"),
    (dict(D=136), "ERR_HEAD_DIM"),
    (dict(scale=0.0), "ERR_SCALE"),
    (dict(scale=float("inf")), "ERR_SCALE"),
    (dict(kn=P), "ERR_NULL_POINTER"),             # k_new without v_new
    (dict(q=0), "ERR_NULL_POINTER"),
    (dict(lens=0), "ERR_NULL_POINTER"),
    (dict(table=0), "ERR_NULL_POINTER"),
    (dict(B=0), "OK"),
    (dict(H=0), "OK"),
    (dict(qs=(256, 64, 2)), "ERR_STRIDE"),
    (dict(qs=(256, 60, 1)), "ERR_STRIDE"),
    (dict(ks=(4096, 1024, 56, 1)), "ERR_STRIDE"),  # rows shorter than the head dim
    (dict(vs=(4096, 1020, 64, 1)), "ERR_STRIDE"),
    (dict(vs=(4096, 1024, 64, 2)), "ERR_STRIDE"),
    (dict(os=(64, 64, 1)), "ERR_STRIDE"),          # rows of O over one another
    (dict(ts=-8), "ERR_STRIDE"),
    (dict(kn=P, vn=P, kns=(256, 63, 1)), "ERR_STRIDE"),
    (dict(q=P + 8), "ERR_ALIGNMENT"),
    (dict(k=P + 2), "ERR_ALIGNMENT"),
    (dict(lens=P + 2), "ERR_ALIGNMENT"),
    (dict(lse=P + 1), "ERR_ALIGNMENT"),
    (dict(work=P + 8, bytes=64), "ERR_ALIGNMENT"),
    (dict(w=P, ws=(512, 100)), "ERR_STRIDE"),      # sums of two heads over one another
    (dict(M=1 << 27), "ERR_TOO_LARGE"),            # 2^31 rows
    (dict(B=1 << 30, H=16, Hkv=16), "ERR_TOO_LARGE"),
])
def test_decode_paged_refuses(lib, kw, code):
    assert _paged(lib, **kw) == _code(code)


# (A call that its strides pass is refused for its misaligned lengths.)
@pytest.mark.parametrize("strides,apart", [
    ((4096, 1024, 64, 1), True),                   # dense
    ((4096, 64, 256, 1), True),                    # a row's heads together
    ((1024, 10240, 64, 1), True),                  # a head's pages together
    ((8192, 2048, 128, 1), True),                  # K and V rows in turn
    ((0, 1024, 64, 1), False),                     # one page for all
    ((4096, 0, 64, 1), False),                     # one head for all
    ((4032, 1024, 64, 1), False),                  # the last row of a page is the next one's first
    ((1024, 4096, 64, 1), False),                  # ten pages, four of which reach the next head
])
def test_written_pools_hold_rows_apart(lib, strides, apart):
    code = _code("ERR_ALIGNMENT" if apart else "ERR_STRIDE")
    for name in ("ks", "vs"):
        assert _paged(lib, kn=P, vn=P, lens=P + 2, **{name: strides}) == code
        assert _paged(lib, lens=P + 2, **{name: strides}) == _code("ERR_ALIGNMENT")   # read only
        assert _evict(lib, lens=P + 2, pages=10, out=2 * P, **{name: strides}) == code
    assert _paged(lib, kn=P, vn=P, lens=P + 2, pages=1, ks=(0, 1024, 64, 1)) == _code("ERR_ALIGNMENT")


def test_key_weights_workspace(lib):
    size = lib.tfserve_key_weights_workspace
    size.restype = ctypes.c_size_t
    assert size(1, 12, 12, 256, 256, 1) == 0 and size(1, 16, 1, 0, 100, 1) == 0 and size(1, 16, 3, 100, 100, 1) == 0
    assert size(8, 64, 64, 4096, 32768, 1) == 0   # keys enough
    n = size(1, 16, 1, 2930, 2930, 1)
    assert 23 * 128 + 2 * 23 * 512 <= n <= 1 << 20
    assert size(1, 16, 1, 2930, 2930, 0) >= n // 2 and n == _C.key_weights_workspace(1, 16, 1, 2930, 2930, True)


def test_decode_paged_workspace(lib):
    f = lib.tfserve_decode_paged_workspace
    f.restype = ctypes.c_size_t
    assert f(1, 12, 12, 16, 4, 64, 0) == 0                          # too short to be divided
    a, b = f(1, 12, 12, 16, 128, 64, 0), f(1, 12, 12, 16, 128, 64, 1)
    assert 0 < a < b and b - a >= 12 * 2048 * 4                     # a score for every head and row
    assert f(200, 32, 32, 64, 64, 64, 0) == 0                       # sequences enough to fill the device
    for bad in ((-1, 4, 4, 16, 8, 64), (2, 4, 3, 16, 8, 64), (2, 4, 4, 0, 8, 64), (2, 4, 4, 16, 8, 60),
                (0, 4, 4, 16, 8, 64), (2, 4, 4, 16, 0, 64)):
        assert f(*bad, 1) == 0
    assert _C.decode_paged_workspace(1, 12, 12, 16, 128, 64, True) == b


def test_workspaces_of_sizes_that_are_refused(lib):
    """Sizes that a call refuses as too large ask for no workspace (nothing is allocated before the refusal)."""
    f, g = lib.tfserve_decode_paged_workspace, lib.tfserve_key_weights_workspace
    f.restype = g.restype = ctypes.c_size_t
    top = 2 ** 31 - 1
    for B, H, H_kv, page, M in ((1, 4, 4, 1, top), (1, 4, 4, 2 ** 20, 2 ** 12), (70000, 4, 4, 16, 8), (top, top, 1, 16, 8)):
        assert f(B, H, H_kv, page, M, 64, 1) == 0
        assert _paged(lib, B=B, H=H, Hkv=H_kv, page=page, M=M) == _code("ERR_TOO_LARGE")
    for H, N_q, N_k in ((16, top, 100), (16, top - 63, 100), (2 ** 20, 2 ** 30, 100), (16, 700, top)):
        assert g(1, H, 1, N_q, N_k, 0) == 0
        assert _weights(lib, B=1, H=H, Hkv=1, Nq=N_q, Nk=N_k) == _code("ERR_TOO_LARGE")


def _weights(lib, **kw):
    a = dict(q=P, qs=(6400, 64, 640, 1), k=P, ks=(6400, 64, 640, 1), lse=P, ls=(1000, 10), out=P, os=(1000, 20), B=2,
             H=10, Hkv=10, Nq=10, Nk=20, D=64, dtype=0, scale=0.125, causal=1, first=0, work=0, bytes=0)
    a.update(kw)
    return lib.tfserve_key_weights(
        _ptr(a["q"]), _strides(*a["qs"]), _ptr(a["k"]), _strides(*a["ks"]), _ptr(a["lse"]), _strides(*a["ls"]),
        _ptr(a["out"]), _strides(*a["os"]), a["B"], a["H"], a["Hkv"], a["Nq"], a["Nk"], a["D"], a["dtype"],
        ctypes.c_float(a["scale"]), a["causal"], I64(a["first"]), _ptr(a["work"]),
        ctypes.c_size_t(a["bytes"]), _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), "ERR_DTYPE"),
    (dict(Nq=-1), "ERR_BAD_SHAPE"),
    (dict(first=-1), "ERR_BAD_SHAPE"),
    (dict(H=15), "ERR_BAD_SHAPE"),
    (dict(D=12), "ERR_HEAD_DIM"),
    (dict(scale=-1.0), "ERR_SCALE"),
    (dict(causal=2), "ERR_CAUSAL_FLAG"),
    (dict(work=P + 8, bytes=1 << 20), "ERR_ALIGNMENT"),
    (dict(Nk=0), "OK"),
    (dict(B=0), "OK"),
    (dict(k=0), "ERR_NULL_POINTER"),
    (dict(lse=0), "ERR_NULL_POINTER"),
    (dict(qs=(6400, 64, 640, 2)), "ERR_STRIDE"),
    (dict(ks=(6400, 64, 56, 1)), "ERR_STRIDE"),
    (dict(os=(1000, 19)), "ERR_STRIDE"),
    (dict(ls=(-1000, 10)), "ERR_STRIDE"),
    (dict(q=P + 4), "ERR_ALIGNMENT"),
    (dict(out=P + 2), "ERR_ALIGNMENT"),
    (dict(B=1 << 20), "ERR_TOO_LARGE"),
])
def test_key_weights_refuses(lib, kw, code):
    assert _weights(lib, **kw) == _code(code)


def _evict(lib, **kw):
    a = dict(k=P, ks=(4096, 1024, 64, 1), v=P, vs=(4096, 1024, 64, 1), table=P, ts=8, lens=P, w=P, ws=(512, 128),
             new=P, ns=4, kept=P, out=P, os=(256, 64), B=2, Hkv=4, pages=20, page=16, M=8, M2=4, D=64, budget=64,
             recent=8)
    a.update(kw)
    return lib.tfserve_evict(
        _ptr(a["k"]), _strides(*a["ks"]), _ptr(a["v"]), _strides(*a["vs"]), _ptr(a["table"]), I64(a["ts"]),
        _ptr(a["lens"]), _ptr(a["w"]), _strides(*a["ws"]), _ptr(a["new"]), I64(a["ns"]), _ptr(a["kept"]), _ptr(a["out"]),
        _strides(*a["os"]), a["B"], a["Hkv"], a["pages"], a["page"], a["M"], a["M2"], a["D"], a["budget"], a["recent"],
        _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(budget=-1), "ERR_BAD_SHAPE"),
    (dict(recent=65), "ERR_BAD_SHAPE"),
    (dict(recent=-1), "ERR_BAD_SHAPE"),
    (dict(budget=65), "ERR_BAD_SHAPE"),            # four new pages hold 64 rows
    (dict(pages=0), "ERR_BAD_SHAPE"),
    (dict(page=0), "ERR_BAD_SHAPE"),
    (dict(D=20), "ERR_HEAD_DIM"),
    (dict(B=0), "OK"),
    (dict(budget=0, recent=0), "OK"),
    (dict(k=0), "ERR_NULL_POINTER"),
    (dict(kept=0), "ERR_NULL_POINTER"),
    (dict(new=0), "ERR_NULL_POINTER"),
    (dict(w=0), "ERR_NULL_POINTER"),
    (dict(ks=(4096, 1024, 48, 1)), "ERR_STRIDE"),
    (dict(ns=3), "ERR_STRIDE"),                    # new tables over one another
    (dict(os=(256, 63)), "ERR_STRIDE"),
    (dict(out=P, os=(1024, 128)), "ERR_STRIDE"),   # the sums themselves at other strides
    (dict(v=P + 4), "ERR_ALIGNMENT"),
    (dict(out=P + 2), "ERR_ALIGNMENT"),
    (dict(M=1 << 27), "ERR_TOO_LARGE"),
    (dict(B=70000), "ERR_TOO_LARGE"),
])
def test_evict_refuses(lib, kw, code):
    if "os" not in kw:
        kw = dict(kw, out=kw.get("out", 2 * P))
    assert _evict(lib, **kw) == _code(code)


def _penalize(lib, **kw):
    a = dict(x=P, xs=100, y=2 * P, ys=100, kind=2, t=P, tb=8, ts=10, n=0, reps=0, rep=1.1, press=0, pres=0.0, freqs=0,
             freq=0.0, bias=0, bs=0, allowed=0, als=0, B=2, V=100, T=10)
    a.update(kw)
    f = ctypes.c_float
    return lib.tfserve_penalize(
        _ptr(a["x"]), I64(a["xs"]), _ptr(a["y"]), I64(a["ys"]), a["kind"], _ptr(a["t"]), a["tb"], I64(a["ts"]),
        _ptr(a["n"]), _ptr(a["reps"]), f(a["rep"]), _ptr(a["press"]), f(a["pres"]), _ptr(a["freqs"]), f(a["freq"]),
        _ptr(a["bias"]), I64(a["bs"]), _ptr(a["allowed"]), I64(a["als"]), a["B"], a["V"], a["T"], _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(kind=3), "ERR_DTYPE"),
    (dict(tb=2), "ERR_DTYPE"),
    (dict(T=-1), "ERR_BAD_SHAPE"),
    (dict(T=2 ** 31 - 300), "ERR_TOO_LARGE"),   # a loop's step past the last token passes 2^31
    (dict(rep=0.0), "ERR_SCALE"),
    (dict(rep=float("nan")), "ERR_SCALE"),
    (dict(pres=float("inf")), "ERR_SCALE"),
    (dict(V=0), "OK"),
    (dict(B=0), "OK"),
    (dict(x=0), "ERR_NULL_POINTER"),
    (dict(t=0), "ERR_NULL_POINTER"),
    (dict(ys=99), "ERR_STRIDE"),
    (dict(xs=-100), "ERR_STRIDE"),
    (dict(y=P, xs=200), "ERR_STRIDE"),             # in place at another stride
    (dict(x=P + 2), "ERR_ALIGNMENT"),
    (dict(t=P + 4), "ERR_ALIGNMENT"),
    (dict(bias=P + 2), "ERR_ALIGNMENT"),
    (dict(B=70000), "ERR_TOO_LARGE"),
])
def test_penalize_refuses(lib, kw, code):
    assert _penalize(lib, **kw) == _code(code)


# ---------------------------------------------------------------------------------------
# The Python functions' own checks, with tensors that only say that they are on a device.


class _Dev(torch.Tensor):
    """A CPU tensor that calls itself a device's."""

    is_cuda = True

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        with torch._C.DisableTorchFunctionSubclass():
            return func(*args, **(kwargs or {}))


def _dev(shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Dev)


I32 = torch.int32


def _paged_args(**kw):
    a = dict(q=_dev((2, 4, 64)), k=_dev((5, 2, 16, 64)), v=_dev((5, 2, 16, 64)), table=_dev((2, 3), I32),
             lens=_dev((2,), I32))
    a.update(kw)
    return [a.pop(n) for n in ("q", "k", "v", "table", "lens")], a


@pytest.mark.parametrize("kw,match", [
    (dict(k=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)), "k_pages must be a CUDA tensor"),
    (dict(k=_dev((5, 2, 16, 64), torch.float32)), "Unsupported tensor dtype"),
    (dict(v=_dev((5, 2, 16, 64), torch.float16)), "v_pages must have dtype"),
    (dict(v=_dev((4, 2, 16, 64))), "v_pages must have shape"),
    (dict(k=_dev((5, 2, 64))), "must be .P, H_kv, page, D."),
    (dict(k=_dev((5, 2, 64, 16)).transpose(2, 3).as_subclass(_Dev)), "dense in its last dimension"),
    (dict(k=_dev((5, 2, 16, 60)), v=_dev((5, 2, 16, 60))), "head_dim must be a multiple of 8"),
    (dict(k=_dev((5, 2, 0, 64)), v=_dev((5, 2, 0, 64))), "a page holds at least one row"),
    (dict(q=_dev((2, 3, 64))), "must be a multiple of the cache's 2"),
    (dict(q=_dev((2, 4, 1, 64))), "q must be"),
    (dict(q=_dev((2, 4, 32))), "q must have shape"),
    (dict(q=_dev((2, 4, 64), torch.float16)), "q must have dtype"),
    (dict(table=_dev((2, 3), torch.int64)), "page_table must be int32"),
    (dict(table=_dev((3, 3), I32)), "page_table must be int32 of shape"),
    (dict(table=_dev((3, 2), I32).t().as_subclass(_Dev)), "page_table must be on"),
    (dict(lens=_dev((3,), I32)), "cache_seqlens must be int32"),
    (dict(k_new=_dev((2, 2, 64))), "must be given together"),
    (dict(k_new=_dev((2, 4, 64)), v_new=_dev((2, 4, 64))), "k_new must have shape"),
    (dict(out=_dev((2, 4, 32))), "out must have shape"),
    (dict(key_weights=_dev((2, 2, 47), torch.float32)), "key_weights must be float32 of shape"),
    (dict(key_weights=_dev((2, 2, 48), torch.float16)), "key_weights must be float32"),
    (dict(workspace=torch.zeros(8, dtype=torch.uint8)), "workspace must be a contiguous tensor"),
])
def test_decode_paged_python_refuses(kw, match):
    args, kw = _paged_args(**kw)
    with pytest.raises(RuntimeError, match=match):
        fa.decode_paged(*args, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16)), "q must be a CUDA tensor"),
    (dict(k=_dev((1, 2, 8, 64), torch.float16)), "k must have dtype"),
    (dict(k=_dev((2, 2, 8, 64))), "k must have shape"),
    (dict(k=_dev((1, 3, 8, 64))), "must be a multiple of k's 3"),
    (dict(q=_dev((1, 4, 8, 20)), k=_dev((1, 2, 8, 20))), "head_dim must be a multiple of 8"),
    (dict(lse=_dev((1, 4, 9), torch.float32)), "lse must be float32 of shape"),
    (dict(lse=_dev((1, 4, 8), torch.float16)), "lse must be float32"),
    (dict(first_query=-1), "first_query must not be negative"),
    (dict(out=_dev((1, 2, 9), torch.float32)), "out must have shape"),
    (dict(out=_dev((1, 4, 8), torch.float32)), "out must be float32 of shape"),
])
def test_key_weights_python_refuses(kw, match):
    a = dict(q=_dev((1, 4, 8, 64)), k=_dev((1, 2, 8, 64)), lse=_dev((1, 4, 8), torch.float32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.key_weights(a.pop("q"), a.pop("k"), a.pop("lse"), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(lens=_dev((2, 1), I32)), "cache_seqlens must be int32"),
    (dict(table=_dev((3, 3), I32)), "page_table must be int32"),
    (dict(new=_dev((2, 2), torch.int64)), "new_page_table must be int32"),
    (dict(w=_dev((2, 2, 40), torch.float32)), "key_weights must be float32 of shape"),
    (dict(budget=33), "do not hold"),
    (dict(budget=8, recent=9), "recent must be between"),
    (dict(weights_out=_dev((2, 2, 31), torch.float32)), "weights_out must be float32"),
])
def test_evict_python_refuses(kw, match):
    a = dict(k=_dev((9, 2, 16, 64)), v=_dev((9, 2, 16, 64)), table=_dev((2, 3), I32), lens=_dev((2,), I32),
             w=_dev((2, 2, 48), torch.float32), new=_dev((2, 2), I32), budget=32)
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.evict(*[a.pop(n) for n in ("k", "v", "table", "lens", "w", "new", "budget")], **a)


@pytest.mark.parametrize("kw,match", [
    (dict(logits=torch.zeros(2, 40)), "logits must be a CUDA tensor"),
    (dict(logits=_dev((2, 40), torch.float64)), "Unsupported tensor dtype"),
    (dict(logits=_dev((40,), torch.float32)), "logits must be"),
    (dict(tokens=_dev((2, 5), torch.int16)), "tokens must be int32 or int64"),
    (dict(tokens=_dev((3, 5), torch.int64)), "tokens must be int32 or int64 of shape"),
    (dict(tokens=None, lengths=_dev((2,), I32)), "lengths needs tokens"),
    (dict(lengths=_dev((2,), torch.int64)), "lengths must be a contiguous int32"),
    (dict(repetition=0.0), "repetition must be finite and positive"),
    (dict(presence=float("nan")), "presence must be finite"),
    (dict(frequency=_dev((3,), torch.float32)), "frequency must be a number or"),
    (dict(bias=_dev((2, 41), torch.float32)), "bias must be"),
    (dict(bias=_dev((40,), torch.float16)), "bias must be"),
    (dict(allowed=_dev((2, 1), I32)), "allowed must be"),
    (dict(out=_dev((2, 40), torch.float16)), "out must be"),
])
def test_penalize_logits_python_refuses(kw, match):
    a = dict(logits=_dev((2, 40), torch.float32), tokens=_dev((2, 5), torch.int64))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.penalize_logits(a.pop("logits"), a.pop("tokens"), **a)


class _OnDevice0(_Dev):
    def get_device(self):
        return 0


@pytest.mark.parametrize("op", ["decode_paged", "key_weights"])
def test_workspace_lives_until_the_launch(monkeypatch, op):
    """Another thread's call on the same stream may replace the kept workspace by a larger one before this call
    launches: the buffer whose address the launch gets is still held then."""
    from custom_flash_attn import serving

    kept, first, launched = {}, [], []

    def make(dev, nbytes):
        buffer = kept["it"] = torch.empty(nbytes, dtype=torch.uint8)
        first.append(weakref.ref(buffer))
        return buffer

    def launch(index, fn, *args):
        kept["it"] = None   # (what the other thread does)
        launched.append(args)
        assert first[0]() is not None, "the workspace was let go before the launch"
        assert args[-2:] == (first[0]().data_ptr(), first[0]().numel())

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(serving, "_current_stream", lambda index: 7)
    monkeypatch.setattr(serving, "_decode_workspace", make)
    monkeypatch.setattr(serving, "_launch_on", launch)
    t = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype).as_subclass(_OnDevice0)  # noqa: E731
    if op == "decode_paged":
        fa.decode_paged(t(1, 4, 64), t(3, 2, 16, 64), t(3, 2, 16, 64), t(1, 100, dtype=I32), t(1, dtype=I32),
                        key_weights=t(1, 2, 1600, dtype=torch.float32))
    else:
        fa.key_weights(t(1, 16, 700, 64), t(1, 1, 700, 64), t(1, 16, 700, dtype=torch.float32))
    assert len(launched) == len(first) == 1
