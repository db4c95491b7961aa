"""CPU-side tests of the boundary of the operators around a paged cache (include/tfgfa_pages.h): every refusal of the C
ABI and of the Python functions, the sizes of workspaces, and a Rotary's frequencies.  No kernel is launched: argument
checks come before any HIP call, and every call here fails them or has nothing to do."""
import ctypes
import math
import os
import re
from fractions import Fraction

import pytest
import torch

import custom_flash_attn as fa
from custom_flash_attn import _C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
P = 0x10000  # a pointer that is never dereferenced
I64 = ctypes.c_int64
TOP = 2 ** 31 - 1


def _code(name):
    return int(re.search(rf"#define\s+TFGFA_{name}\s+(-?\d+)", open(os.path.join(INCLUDE, "tfgfa.h")).read()).group(1))


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(fa.library_path())


def test_library_exports_the_entry_points(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INCLUDE, "tfgfa_pages.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(tfpages_\w+)\s*\(", text)))
    assert names == ["tfpages_append", "tfpages_attend", "tfpages_attend_workspace", "tfpages_decode_shared",
                     "tfpages_decode_shared_workspace", "tfpages_rotate"]
    assert all(hasattr(lib, n) for n in names) and lib.tfgfa_abi_version() >= 11


def _ptr(x):
    return ctypes.c_void_p(x)


def _st(v):
    return (I64 * len(v))(*v)


F = ctypes.c_float


def _rotate(lib, **kw):
    a = dict(q=P, qs=(2560, 64, 256, 1), qo=2 * P, qos=(2560, 64, 256, 1), H=4, k=0, ks=(0, 0, 0, 1), ko=0, kos=(0, 0, 0, 1),
             Hkv=0, pos=P, pb=4, ps=(0, 1), first=0, turns=P, rot=64, inter=0, m=1.0, tr=0, B=2, N=10, D=64, dtype=0)
    a.update(kw)
    return lib.tfpages_rotate(
        _ptr(a["q"]), _st(a["qs"]), _ptr(a["qo"]), _st(a["qos"]), a["H"], _ptr(a["k"]), _st(a["ks"]), _ptr(a["ko"]),
        _st(a["kos"]), a["Hkv"], _ptr(a["pos"]), a["pb"], _st(a["ps"]), I64(a["first"]), _ptr(a["turns"]), a["rot"],
        a["inter"], F(a["m"]), a["tr"], a["B"], a["N"], a["D"], a["dtype"], _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), "ERR_DTYPE"),
    (dict(pb=2), "ERR_DTYPE"),
    (dict(B=-1), "ERR_BAD_SHAPE"),
    (dict(inter=2), "ERR_BAD_SHAPE"),
    (dict(tr=-1), "ERR_BAD_SHAPE"),
    (dict(rot=63), "ERR_HEAD_DIM"),
    (dict(rot=66), "ERR_HEAD_DIM"),
    (dict(D=130, rot=2), "ERR_HEAD_DIM"),
    (dict(m=0.0), "ERR_SCALE"),
    (dict(m=float("nan")), "ERR_SCALE"),
    (dict(B=0), "OK"),
    (dict(N=0), "OK"),
    (dict(H=0), "OK"),
    (dict(B=TOP, N=2), "ERR_TOO_LARGE"),
    (dict(B=1 << 14, N=(1 << 13) + 1), "ERR_TOO_LARGE"),   # past 2^27 tokens
    (dict(q=0), "ERR_NULL_POINTER"),
    (dict(turns=0), "ERR_NULL_POINTER"),
    (dict(Hkv=2), "ERR_NULL_POINTER"),
    (dict(qs=(2560, 64, 256, 2)), "ERR_STRIDE"),
    (dict(qs=(-2560, 64, 256, 1)), "ERR_STRIDE"),
    (dict(qos=(2560, 0, 256, 1)), "ERR_STRIDE"),       # heads of the output over one another
    (dict(qos=(2560, 32, 256, 1)), "ERR_STRIDE"),
    (dict(qo=P, qos=(2560, 640, 64, 1)), "ERR_STRIDE"),  # in place in another layout
    (dict(q=P + 1), "ERR_ALIGNMENT"),
    (dict(q=P + 2, dtype=2), "ERR_ALIGNMENT"),
    (dict(pos=P + 2), "ERR_ALIGNMENT"),
    (dict(pos=P + 4, pb=8), "ERR_ALIGNMENT"),
    (dict(turns=P + 4), "ERR_ALIGNMENT"),
])
def test_rotate_refuses(lib, kw, code):
    assert _rotate(lib, **kw) == _code(code)


def _append(lib, **kw):
    a = dict(k=P, ks=(1280, 64, 128, 1), v=P, vs=(1280, 64, 128, 1), kp=P, kps=(4096, 1024, 64, 1), vp=P,
             vps=(4096, 1024, 64, 1), table=P, ts=8, lens=P, new=0, pos=0, q=0, qs=(2560, 64, 256, 1), qo=0,
             qos=(2560, 64, 256, 1), pad=1, turns=P, rot=64, inter=0, m=1.0, B=2, H=4, Hkv=2, N=10, pages=10, page=16, M=8,
             D=64, dtype=0)
    a.update(kw)
    return lib.tfpages_append(
        _ptr(a["k"]), _st(a["ks"]), _ptr(a["v"]), _st(a["vs"]), _ptr(a["kp"]), _st(a["kps"]), _ptr(a["vp"]), _st(a["vps"]),
        _ptr(a["table"]), I64(a["ts"]), _ptr(a["lens"]), _ptr(a["new"]), _ptr(a["pos"]), _ptr(a["q"]), _st(a["qs"]),
        _ptr(a["qo"]), _st(a["qos"]), a["pad"], _ptr(a["turns"]), a["rot"], a["inter"], F(a["m"]), a["B"], a["H"], a["Hkv"],
        a["N"], a["pages"], a["page"], a["M"], a["D"], a["dtype"], _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), "ERR_DTYPE"),
    (dict(N=-1), "ERR_BAD_SHAPE"),
    (dict(page=0), "ERR_BAD_SHAPE"),
    (dict(M=-1), "ERR_BAD_SHAPE"),
    (dict(pages=-1), "ERR_BAD_SHAPE"),
    (dict(D=60, rot=60), "ERR_HEAD_DIM"),
    (dict(rot=65), "ERR_HEAD_DIM"),
    (dict(m=float("inf")), "ERR_SCALE"),
    (dict(q=P), "ERR_NULL_POINTER"),
    (dict(qo=P), "ERR_NULL_POINTER"),
    (dict(B=0), "OK"),
    (dict(N=0), "OK"),
    (dict(Hkv=0), "OK"),
    (dict(Hkv=0, q=P, qo=P), "ERR_BAD_SHAPE"),
    (dict(B=TOP, N=2), "ERR_TOO_LARGE"),
    (dict(B=1 << 14, N=(1 << 13) + 1), "ERR_TOO_LARGE"),   # past 2^27 tokens
    (dict(M=1 << 27), "ERR_TOO_LARGE"),
    (dict(k=0), "ERR_NULL_POINTER"),
    (dict(lens=0), "ERR_NULL_POINTER"),
    (dict(table=0), "ERR_NULL_POINTER"),
    (dict(turns=0), "ERR_NULL_POINTER"),
    (dict(ks=(1280, 64, 127, 1)), "ERR_STRIDE"),
    (dict(vs=(1280, 64, 56, 1)), "ERR_STRIDE"),
    (dict(kps=(0, 1024, 64, 1)), "ERR_STRIDE"),        # one page for all
    (dict(vps=(4096, 1024, 32, 1)), "ERR_STRIDE"),
    (dict(ts=-1), "ERR_STRIDE"),
    (dict(q=P, qo=2 * P, qos=(2560, 0, 256, 1)), "ERR_STRIDE"),
    (dict(q=P, qo=P, qos=(2560, 640, 64, 1)), "ERR_STRIDE"),
    (dict(kp=P + 8), "ERR_ALIGNMENT"),
    (dict(q=P + 8, qo=P), "ERR_ALIGNMENT"),
    (dict(lens=P + 2), "ERR_ALIGNMENT"),
    (dict(new=P + 1), "ERR_ALIGNMENT"),
    (dict(pos=P + 3), "ERR_ALIGNMENT"),
    (dict(turns=P + 4), "ERR_ALIGNMENT"),
])
def test_append_refuses(lib, kw, code):
    assert _append(lib, **kw) == _code(code)


def _attend(lib, **kw):
    a = dict(q=P, qs=(2560, 64, 256, 1), k=P, ks=(4096, 1024, 64, 1), v=P, vs=(4096, 1024, 64, 1), table=P, ts=8, lens=P,
             new=0, o=P, os=(2560, 64, 256, 1), lse=0, pad=1, causal=1, B=2, H=4, Hkv=2, N=10, pages=10, page=16, M=8, D=64,
             dtype=0, scale=0.125, work=0, bytes=0)
    a.update(kw)
    return lib.tfpages_attend(
        _ptr(a["q"]), _st(a["qs"]), _ptr(a["k"]), _st(a["ks"]), _ptr(a["v"]), _st(a["vs"]), _ptr(a["table"]), I64(a["ts"]),
        _ptr(a["lens"]), _ptr(a["new"]), _ptr(a["o"]), _st(a["os"]), _ptr(a["lse"]), a["pad"], a["causal"], a["B"], a["H"],
        a["Hkv"], a["N"], a["pages"], a["page"], a["M"], a["D"], a["dtype"], F(a["scale"]), _ptr(a["work"]),
        ctypes.c_size_t(a["bytes"]), _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), "ERR_DTYPE"),
    (dict(H=3), "ERR_BAD_SHAPE"),
    (dict(Hkv=0), "ERR_BAD_SHAPE"),
    (dict(N=-1), "ERR_BAD_SHAPE"),
    (dict(page=0), "ERR_BAD_SHAPE"),
    (dict(pages=0), "ERR_BAD_SHAPE"),
    (dict(D=136), "ERR_HEAD_DIM"),
    (dict(scale=0.0), "ERR_SCALE"),
    (dict(causal=2), "ERR_CAUSAL_FLAG"),
    (dict(B=0), "OK"),
    (dict(H=0), "OK"),
    (dict(N=0), "OK"),
    (dict(M=1 << 27), "ERR_TOO_LARGE"),
    (dict(N=TOP), "ERR_TOO_LARGE"),
    (dict(B=TOP), "ERR_TOO_LARGE"),
    (dict(B=1 << 23), "ERR_TOO_LARGE"),                             # 2^24 workgroups of 256 threads
    (dict(ks=(4096, 1024, 1 << 27, 1), page=1), "ERR_ALIGNMENT"),   # (the stride of one row is not taken)
    (dict(ks=(4096, 1024, 1 << 27, 1)), "ERR_TOO_LARGE"),           # 8 rows past 2^30 bytes
    (dict(q=0), "ERR_NULL_POINTER"),
    (dict(lens=0), "ERR_NULL_POINTER"),
    (dict(table=0), "ERR_NULL_POINTER"),
    (dict(qs=(2560, 64, 252, 1)), "ERR_STRIDE"),
    (dict(ks=(4096, 1024, 56, 1)), "ERR_STRIDE"),
    (dict(vs=(4096, 1024, 64, 2)), "ERR_STRIDE"),
    (dict(os=(2560, 0, 256, 1)), "ERR_STRIDE"),
    (dict(ts=-8), "ERR_STRIDE"),
    (dict(v=P + 8), "ERR_ALIGNMENT"),
    (dict(work=P + 4, bytes=1 << 20), "ERR_ALIGNMENT"),
    (dict(lens=P + 1), "ERR_ALIGNMENT"),
    (dict(lse=P + 2), "ERR_ALIGNMENT"),
])
def test_attend_refuses(lib, kw, code):
    assert _attend(lib, **{**dict(lens=P + 2 if code == "ERR_ALIGNMENT" else P), **kw}) == _code(code)


def _shared(lib, **kw):
    a = dict(q=P, qs=(256, 64, 1), k=P, ks=(4096, 1024, 64, 1), v=P, vs=(4096, 1024, 64, 1), pt=P, pts=8, pl=P, table=P, ts=8,
             lens=P, kn=0, kns=(128, 64, 1), vn=0, vns=(128, 64, 1), o=P, os=(256, 64, 1), lse=0, R=2, B=6, H=4, Hkv=2, pages=10,
             page=16, Mp=8, M=8, D=64, dtype=0, scale=0.125, work=P, bytes=1 << 24)
    a.update(kw)
    return lib.tfpages_decode_shared(
        _ptr(a["q"]), _st(a["qs"]), _ptr(a["k"]), _st(a["ks"]), _ptr(a["v"]), _st(a["vs"]), _ptr(a["pt"]), I64(a["pts"]),
        _ptr(a["pl"]), _ptr(a["table"]), I64(a["ts"]), _ptr(a["lens"]), _ptr(a["kn"]), _st(a["kns"]), _ptr(a["vn"]),
        _st(a["vns"]), _ptr(a["o"]), _st(a["os"]), _ptr(a["lse"]), a["R"], a["B"], a["H"], a["Hkv"], a["pages"], a["page"],
        a["Mp"], a["M"], a["D"], a["dtype"], F(a["scale"]), _ptr(a["work"]), ctypes.c_size_t(a["bytes"]), _ptr(0))


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), "ERR_DTYPE"),
    (dict(R=4), "ERR_BAD_SHAPE"),
    (dict(R=0), "ERR_BAD_SHAPE"),
    (dict(R=-1), "ERR_BAD_SHAPE"),
    (dict(H=5), "ERR_BAD_SHAPE"),
    (dict(Mp=-1), "ERR_BAD_SHAPE"),
    (dict(pages=0), "ERR_BAD_SHAPE"),
    (dict(D=4), "ERR_HEAD_DIM"),
    (dict(scale=-1.0), "ERR_SCALE"),
    (dict(kn=P), "ERR_NULL_POINTER"),
    (dict(B=0), "OK"),
    (dict(H=0), "OK"),
    (dict(Mp=1 << 27), "ERR_TOO_LARGE"),
    (dict(M=1 << 27), "ERR_TOO_LARGE"),
    (dict(R=1, B=1 << 23), "ERR_TOO_LARGE"),                 # 2^24 workgroups of 256 threads
    (dict(R=1, B=1 << 22, H=32, Hkv=1), "ERR_TOO_LARGE"),    # and for the join
    (dict(q=0), "ERR_NULL_POINTER"),
    (dict(pl=0), "ERR_NULL_POINTER"),
    (dict(pt=0), "ERR_NULL_POINTER"),
    (dict(table=0), "ERR_NULL_POINTER"),
    (dict(qs=(256, 60, 1)), "ERR_STRIDE"),
    (dict(os=(64, 64, 1)), "ERR_STRIDE"),
    (dict(kn=P, vn=P, ks=(0, 1024, 64, 1)), "ERR_STRIDE"),   # a pool that is written to
    (dict(ts=-1), "ERR_STRIDE"),
    (dict(pts=-1), "ERR_STRIDE"),
    (dict(k=P + 8), "ERR_ALIGNMENT"),
    (dict(pl=P + 2), "ERR_ALIGNMENT"),
    (dict(work=P + 8), "ERR_ALIGNMENT"),
    (dict(bytes=1024), "ERR_SCRATCH"),
    (dict(work=0), "ERR_SCRATCH"),
])
def test_decode_shared_refuses(lib, kw, code):
    assert _shared(lib, **kw) == _code(code)


def test_workspaces(lib):
    f, g = lib.tfpages_attend_workspace, lib.tfpages_decode_shared_workspace
    f.restype = g.restype = ctypes.c_size_t
    assert f(64, 16, 16, 2048, 64, 512, 64) == 0              # rows enough to fill the device
    assert f(1, 12, 12, 4, 16, 8, 64) == 0                    # too few keys to be divided
    a = f(1, 32, 8, 4, 16, 2048, 128)
    assert a >= 8 * 2 * 32 * 131 * 4 and a == _C.attend_workspace(1, 32, 8, 4, 16, 2048, 128)
    for bad in ((-1, 4, 4, 4, 16, 8, 64), (2, 4, 3, 4, 16, 8, 64), (2, 4, 4, 4, 0, 8, 64), (2, 4, 4, 4, 16, 8, 60),
                (0, 4, 4, 4, 16, 8, 64), (2, 4, 4, 0, 16, 8, 64), (1, 4, 4, 4, 1, TOP, 64), (1, 4, 4, TOP, 16, 8, 64)):
        assert f(*bad) == 0
    b = g(1, 64, 32, 8, 128, 256, 4, 128)
    assert b >= 64 * 32 * 131 * 4 and b == _C.decode_shared_workspace(1, 64, 32, 8, 128, 256, 4, 128)
    for bad in ((0, 4, 4, 4, 16, 8, 8, 64), (3, 4, 4, 4, 16, 8, 8, 64), (1, 4, 4, 3, 16, 8, 8, 64), (1, 0, 4, 4, 16, 8, 8, 64),
                (1, 4, 4, 4, 16, -1, 8, 64), (1, 4, 4, 4, 16, 8, 8, 65), (1, 4, 4, 4, 1, TOP, 8, 64)):
        assert g(*bad) == 0


# ---------------------------------------------------------------------------------------
# Frequencies.


def test_rotary_frequencies():
    r = fa.Rotary(64, device="cpu")
    assert [x for x in r.frequencies] == [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert fa.Rotary(64, scaling="linear", factor=4.0, device="cpu").frequencies[5] == r.frequencies[5] / 4
    b = fa.Rotary(64, scaling="base", factor=4.0, device="cpu").frequencies
    assert b[0] == 1.0 and abs(b[31] / (r.frequencies[31] / 4) - 1) < 1e-12
    c = fa.Rotary(64, scaling="bands", factor=8.0, trained_length=1024, low=1.0, high=32.0, device="cpu").frequencies
    turns = [1024 * x / (2 * math.pi) for x in r.frequencies]
    for i, n in enumerate(turns):
        keep = 1.0 if n >= 32 else 0.0 if n <= 1 else (n - 1) / 31
        assert abs(c[i] / (r.frequencies[i] * (keep + (1 - keep) / 8)) - 1) < 1e-12
    assert c[0] == 1.0 and c[31] == r.frequencies[31] / 8 and any(n > 1 and n < 32 for n in turns)
    # Turns in 2^-64: the nearest integer to the float64 quotient, itself off by 2^-53 of it at most (pi by 2^-54).
    for f, t in zip(r.frequencies, r._turns.tolist()):
        exact = Fraction(f) / (2 * Fraction(math.pi))
        assert abs(Fraction(t % 2 ** 64, 2 ** 64) - exact) <= exact / 2 ** 52 + Fraction(1, 2 ** 65)
    given = fa.Rotary(4, frequencies=torch.tensor([20.0, -0.5]), interleaved=True, device="cpu")
    assert given.frequencies == (20.0, -0.5)
    for f, t in zip(given.frequencies, given._turns.tolist()):
        exact = Fraction(f) / (2 * Fraction(math.pi)) % 1
        assert abs(Fraction(t % 2 ** 64, 2 ** 64) - exact) <= Fraction(4, 2 ** 52)
    assert given.to("cpu")._turns.tolist() == given._turns.tolist() and given.to("cpu").interleaved


@pytest.mark.parametrize("kw,match", [
    (dict(dim=63), "dim must be even"),
    (dict(dim=0), "dim must be even"),
    (dict(dim=130), "dim must be even"),
    (dict(base=0.0), "base must be"),
    (dict(scaling="other"), "scaling must be"),
    (dict(factor=2.0), "factor must be"),
    (dict(scaling="linear", factor=0.0), "factor must be"),
    (dict(scaling="bands", factor=2.0), "trained_length"),
    (dict(scaling="bands", factor=2.0, trained_length=100, low=4.0, high=4.0), "low < high"),
    (dict(magnitude=0.0), "magnitude must be"),
    (dict(frequencies=[1.0]), "frequencies must be 32"),
    (dict(frequencies=[float("inf")] * 32), "frequencies must be 32 finite"),
    (dict(frequencies=[1.0] * 32, scaling="linear"), "no scaling"),
])
def test_rotary_refuses(kw, match):
    kw = dict(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.Rotary(kw.pop("dim", 64), device="cpu", **kw)


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


def _turned_last(shape):
    return _dev(shape).transpose(2, 3).as_subclass(_Dev)


I32 = torch.int32
HF = torch.float16


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(2, 4, 8, 64)), "q must be a CUDA tensor"),
    (dict(q=_dev((2, 4, 8, 64), torch.float64)), "Unsupported tensor dtype"),
    (dict(q=_dev((2, 4, 64))), "q must be 4-D"),
    (dict(q=_turned_last((2, 4, 64, 8))), "dense in its last dimension"),
    (dict(k=_dev((2, 2, 8, 64), HF)), "k must have dtype"),
    (dict(k=_dev((2, 2, 9, 64))), "k must have shape"),
    (dict(q=_dev((2, 4, 8, 136)), k=None), "head_dim must be"),
    (dict(q_out=_dev((2, 4, 8, 32))), "q_out must have the shape"),
    (dict(k=None, k_out=_dev((2, 2, 8, 64))), "k_out must have the shape"),
    (dict(rotary=None), "rotary must be a Rotary"),
    (dict(rotary=fa.Rotary(128, device="cpu")), "rotates 128 dims"),
    (dict(positions=_dev((8,), torch.int16)), "positions must be int32 or int64"),
    (dict(positions=_dev((2,), I32)), "positions must be int32 or int64 of shape"),
    (dict(positions=1.5), "positions must be a tensor or the first"),
])
def test_rotate_python_refuses(kw, match):
    a = dict(q=_dev((2, 4, 8, 64)), k=_dev((2, 2, 8, 64)), positions=0, rotary=fa.Rotary(64, device="cpu"))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.rotate(*[a.pop(n) for n in ("q", "k", "positions", "rotary")], **a)


@pytest.mark.parametrize("kw,match", [
    (dict(k=torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16)), "k must be a CUDA tensor"),
    (dict(k=_dev((2, 2, 64))), "k must be 4-D"),
    (dict(k=_dev((2, 4, 8, 64))), "k must have shape"),
    (dict(v=_dev((2, 2, 7, 64))), "v must have shape"),
    (dict(v=_dev((2, 2, 8, 64), HF)), "v must have dtype"),
    (dict(v=_turned_last((2, 2, 64, 8))), "v must be dense"),
    (dict(v_pages=_dev((4, 2, 16, 64))), "v_pages must have shape"),
    (dict(table=_dev((3, 3), I32)), "page_table must be int32"),
    (dict(lens=_dev((2,), torch.int64)), "cache_seqlens must be int32"),
    (dict(lengths=_dev((3,), I32)), "lengths must be a contiguous int32"),
    (dict(positions=_dev((2,), I32)), "positions needs a rotary"),
    (dict(q=_dev((2, 4, 8, 64))), "q needs a rotary"),
    (dict(q_out=_dev((2, 4, 8, 64))), "q_out needs q"),
    (dict(rotary=fa.Rotary(128, device="cpu")), "rotates 128 dims"),
    (dict(rotary=fa.Rotary(64, device="cpu"), positions=_dev((2, 8), I32)), "positions must be a contiguous int32"),
    (dict(rotary=fa.Rotary(64, device="cpu"), q=_dev((2, 4, 64))), "q must be 4-D"),
    (dict(rotary=fa.Rotary(64, device="cpu"), q=_dev((2, 4, 9, 64))), "q must have shape"),
    (dict(rotary=fa.Rotary(64, device="cpu"), q=_dev((2, 4, 8, 64)), q_out=_dev((2, 2, 8, 64))), "q_out must have shape"),
])
def test_append_paged_python_refuses(kw, match):
    a = dict(k=_dev((2, 2, 8, 64)), v=_dev((2, 2, 8, 64)), k_pages=_dev((5, 2, 16, 64)), v_pages=_dev((5, 2, 16, 64)),
             table=_dev((2, 3), I32), lens=_dev((2,), I32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.append_paged(*[a.pop(n) for n in ("k", "v", "k_pages", "v_pages", "table", "lens")], **a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16)), "q must be a CUDA tensor"),
    (dict(q=_dev((2, 4, 64))), "q must be 4-D"),
    (dict(q=_dev((2, 3, 8, 64))), "must be a multiple of the cache's 2"),
    (dict(q=_dev((2, 4, 8, 32))), "q must have shape"),
    (dict(q=_dev((2, 4, 8, 64), HF)), "q must have dtype"),
    (dict(out=_dev((2, 4, 9, 64))), "out must have shape"),
    (dict(k=_dev((5, 2, 16, 64), torch.float32)), "Unsupported tensor dtype"),
    (dict(table=_dev((3, 3), I32)), "page_table must be int32"),
    (dict(lens=_dev((3,), I32)), "cache_seqlens must be int32"),
    (dict(lengths=_dev((2,), torch.int64)), "lengths must be a contiguous int32"),
    (dict(workspace=torch.zeros(8, dtype=torch.uint8)), "workspace must be a contiguous tensor"),
])
def test_attend_paged_python_refuses(kw, match):
    a = dict(q=_dev((2, 4, 8, 64)), k=_dev((5, 2, 16, 64)), v=_dev((5, 2, 16, 64)), table=_dev((2, 3), I32),
             lens=_dev((2,), I32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.attend_paged(*[a.pop(n) for n in ("q", "k", "v", "table", "lens")], **a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=_dev((6, 4, 1, 64))), "q must be"),
    (dict(q=_dev((6, 3, 64))), "must be a multiple of the cache's 2"),
    (dict(pt=_dev((4, 3), I32)), "a multiple of R"),
    (dict(pt=_dev((3,), I32)), "prefix_table must be int32"),
    (dict(pt=_dev((2, 3), torch.int64)), "prefix_table must be int32"),
    (dict(pl=_dev((6,), I32)), "prefix_lens must be a contiguous int32"),
    (dict(table=_dev((2, 3), I32)), "page_table must be int32"),
    (dict(lens=_dev((2,), I32)), "cache_seqlens must be int32"),
    (dict(k_new=_dev((6, 2, 64))), "must be given together"),
    (dict(k_new=_dev((6, 4, 64)), v_new=_dev((6, 4, 64))), "k_new must have shape"),
    (dict(out=_dev((6, 4, 32))), "out must have shape"),
    (dict(workspace=torch.zeros(8, dtype=torch.uint8)), "workspace must be a contiguous tensor"),
])
def test_decode_shared_python_refuses(kw, match):
    a = dict(q=_dev((6, 4, 64)), k=_dev((5, 2, 16, 64)), v=_dev((5, 2, 16, 64)), pt=_dev((2, 3), I32), pl=_dev((2,), I32),
             table=_dev((6, 3), I32), lens=_dev((6,), I32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        fa.decode_shared(*[a.pop(n) for n in ("q", "k", "v", "pt", "pl", "table", "lens")], **a)


class _OnDevice0(torch.Tensor):
    """A tensor of the CPU that says it is on device 0."""

    is_cuda = True

    def get_device(self):
        return 0


@pytest.mark.parametrize("op", ["attend_paged", "decode_shared"])
def test_workspace_lives_until_the_launch(monkeypatch, op):
    """Another thread's call on the same stream may replace the kept workspace by a larger one before this call launches: the
    buffer whose address the launch gets is still held then."""
    import weakref

    from custom_flash_attn import pages, serving

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
    monkeypatch.setattr(pages, "_launch_on", launch)
    t = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype).as_subclass(_OnDevice0)  # noqa: E731
    i32 = dict(dtype=torch.int32)
    if op == "attend_paged":
        fa.attend_paged(t(1, 4, 3, 64), t(3, 2, 16, 64), t(3, 2, 16, 64), t(1, 1000, **i32), t(1, **i32))
    else:
        fa.decode_shared(t(4, 4, 64), t(3, 2, 16, 64), t(3, 2, 16, 64), t(2, 9, **i32), t(2, **i32), t(4, 2, **i32), t(4, **i32))
    assert len(launched) == len(first) == 1
