"""The operators around a paged KV cache (include/tfgfa_pages.h) on torch tensors: rotary positions, new tokens' keys
and values into the pages, attention of several new tokens over them, and a decode step for sequences that share a
prefix.

The reference's model has learned positions and keeps no cache (src/py/model_inference.py:166-228); nothing here has
a counterpart in it.  The functions check their arguments (RuntimeError, before anything is launched), launch on the
current stream of the tensors' device and do not synchronise.  :func:`rotate` has a gradient; the others are inference
operators, whose results carry none.  Tensors of the caller's that are written (outputs, pools) count a version, as by torch's
operators in place, so that a backward pass that needs their old values raises; those that require a gradient are refused
where gradients are recorded.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _C, _check_vec, _DTYPES, MAX_HEAD_DIM, _launch_on
from .serving import (_accepts_pages, _check_pages, _check_seqlens, _check_table, _extent, _is_seqlens, _is_table,
                      _workspace)

_NONE, _NONE3 = (0, (0, 0, 0, 0)), (0, (0, 0, 0))
_ROTATED = {torch.bfloat16: _C.DTYPE_BF16, torch.float16: _C.DTYPE_F16, torch.float32: _C.DTYPE_F32}
_INTS = (torch.int32, torch.int64)

# Whether a function transform is active, and the forward-mode level (a torch without them has neither).
_transform = getattr(getattr(torch._C, "_functorch", None), "peek_interpreter_stack", lambda: None)


def _check_written(*tensors) -> None:
    """Tensors that a call writes beside autograd (None: not given)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("a tensor that is written requires a gradient, which is not differentiable: call under "
                                   "torch.no_grad() or give another")


def _view(t):
    return _NONE if t is None else (t.data_ptr(), t.stride())


class Rotary:
    """A model's rotary positions: of each head's first ``dim`` dims (even, the whole head or a part of it) pair i is
    turned by ``position * frequencies[i]`` radians.  Pairs are dims (i, i + dim / 2), or with ``interleaved`` (2i, 2i + 1).

    Frequencies are ``base ** (-2 i / dim)``, for contexts longer than the trained ones scaled by ``factor``:
      * ``scaling="linear"``: divided by it;
      * ``scaling="base"``: of base ``base * factor ** (dim / (dim - 2))``, which divides the last by it and keeps the first;
      * ``scaling="bands"``: those that turn at least ``high`` times within ``trained_length`` positions are kept, those
        that turn at most ``low`` times divided, those between mixed in proportion to their turns;
    or ``frequencies`` (dim / 2 numbers, radians a position) gives them.  ``magnitude`` multiplies what is rotated.
    They are kept on ``device`` as 64-bit fractions of a turn, so that an angle is exact at any position.
    """

    def __init__(self, dim: int, base: float = 10000.0, *, interleaved: bool = False, scaling: str | None = None,
                 factor: float = 1.0, trained_length: int | None = None, low: float = 1.0, high: float = 32.0,
                 magnitude: float = 1.0, frequencies=None, device="cuda"):
        if not (isinstance(dim, int) and 2 <= dim <= MAX_HEAD_DIM and dim % 2 == 0):
            raise RuntimeError(f"dim must be even, in [2, {MAX_HEAD_DIM}], got {dim}")
        if not (math.isfinite(magnitude) and magnitude > 0):
            raise RuntimeError(f"magnitude must be finite and positive, got {magnitude}")
        if frequencies is not None:
            if scaling is not None:
                raise RuntimeError("frequencies are given as they are: no scaling beside them")
            f = [float(x) for x in frequencies]
            if len(f) != dim // 2 or not all(math.isfinite(x) for x in f):
                raise RuntimeError(f"frequencies must be {dim // 2} finite numbers")
        else:
            if not (math.isfinite(base) and base > 0):
                raise RuntimeError(f"base must be finite and positive, got {base}")
            if scaling not in (None, "linear", "base", "bands"):
                raise RuntimeError(f"scaling must be None, 'linear', 'base' or 'bands', got {scaling!r}")
            if not (math.isfinite(factor) and factor > 0) or (scaling is None and factor != 1.0):
                raise RuntimeError(f"factor must be finite and positive, and 1 without scaling, got {factor}")
            try:
                if scaling == "base" and dim > 2:
                    base = base * factor ** (dim / (dim - 2))
                f = [base ** (-2 * i / dim) for i in range(dim // 2)] if 0 < base < math.inf else [math.inf]
            except OverflowError:
                f = [math.inf]
            if scaling == "linear":
                f = [x / factor for x in f]
            elif scaling == "bands":
                if trained_length is None or not trained_length > 0 or not 0 <= low < high < math.inf:
                    raise RuntimeError("scaling='bands' needs a positive trained_length and 0 <= low < high, got "
                                       f"{trained_length}, {low} and {high}")
                for i, x in enumerate(f):
                    keep = min(1.0, max(0.0, (trained_length * x / (2 * math.pi) - low) / (high - low)))
                    f[i] = x / factor * (1 - keep) + x * keep
            if not all(math.isfinite(x) for x in f):
                raise RuntimeError(f"base and factor give frequencies past float64's range, got {base} and {factor}")
        self.dim, self.interleaved, self.magnitude, self.frequencies = dim, bool(interleaved), float(magnitude), tuple(f)
        self._turns = torch.tensor([_turn(x) for x in f], dtype=torch.int64).to(device)

    def to(self, device) -> "Rotary":
        """The same on another device."""
        return Rotary(self.dim, interleaved=self.interleaved, magnitude=self.magnitude, frequencies=self.frequencies,
                      device=device)


def _turn(frequency: float) -> int:
    """The frequency as turns in 2^-64, modulo a turn, as a signed 64-bit integer (the nearest to the float64 quotient)."""
    n = round(math.fmod(frequency / (2 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64
    return n - 2 ** 64 if n >= 2 ** 63 else n


def _is_rotary(rotary, index: int, D: int) -> bool:
    return type(rotary) is Rotary and rotary._turns.get_device() == index and rotary.dim <= D


def _check_rotary(rotary, dev, D: int) -> None:
    if not isinstance(rotary, Rotary):
        raise RuntimeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    if rotary._turns.device != dev:
        raise RuntimeError(f"rotary must be on {dev}, got {rotary._turns.device}")
    if rotary.dim > D:
        raise RuntimeError(f"rotary rotates {rotary.dim} dims of a head of {D}")


def _are_positions(p, B: int, N: int, index: int) -> bool:
    return p.dtype in _INTS and p.get_device() == index and p.shape in ((N,), (B, N), (1, N))


def _is_first(p) -> bool:
    return type(p) is int and -2 ** 63 <= p < 2 ** 63


def _accepts_rotate(q, k, positions, rotary, outs) -> bool:
    """Everything _check_rotate checks, as one test."""
    qs, index, dtype = q.shape, q.get_device(), q.dtype
    if not (index >= 0 and q.is_cuda and dtype in _ROTATED and len(qs) == 4 and 1 <= qs[3] <= MAX_HEAD_DIM
            and (q.stride(3) == 1 or qs[3] == 1) and _is_rotary(rotary, index, qs[3])):
        return False
    if k is not None:
        ks = k.shape
        if not (k.dtype is dtype and k.get_device() == index and len(ks) == 4 and ks[0] == qs[0] and ks[2] == qs[2]
                and ks[3] == qs[3] and (k.stride(3) == 1 or qs[3] == 1)):
            return False
    for x, out in zip((q, k), outs):
        if out is not None and not (x is not None and out.shape == x.shape and out.dtype is dtype
                                    and out.get_device() == index and (out.stride(3) == 1 or qs[3] == 1)):
            return False
    return _is_first(positions) or (isinstance(positions, torch.Tensor) and _are_positions(positions, qs[0], qs[2], index))


def _check_rotate(q, k, positions, rotary, outs) -> None:
    for x, n in ((q, "q"), (k, "k"), (outs[0], "q_out"), (outs[1], "k_out")):
        if x is None:
            continue
        if not x.is_cuda:
            raise RuntimeError(f"{n} must be a CUDA tensor")
        if x.dtype not in _ROTATED:
            raise RuntimeError("Unsupported tensor dtype. Use float32, bfloat16 or float16.")
        if x.dim() != 4:
            raise RuntimeError(f"{n} must be 4-D (batch, heads, seq_len, head_dim), got shape {tuple(x.shape)}")
        if x.stride(3) != 1 and x.shape[3] > 1:
            raise RuntimeError(f"{n} must be dense in its last dimension (stride 1), got strides {x.stride()}")
        if x.dtype != q.dtype:
            raise RuntimeError(f"{n} must have dtype {q.dtype}, got {x.dtype}")
        if x.device != q.device:
            raise RuntimeError(f"{n} must be on {q.device}, got {x.device}")
    B, _, N, D = q.shape
    if not 1 <= D <= MAX_HEAD_DIM:
        raise RuntimeError(f"head_dim must be in [1, {MAX_HEAD_DIM}], got {D}")
    if k is not None and (k.shape[0], k.shape[2], k.shape[3]) != (B, N, D):
        raise RuntimeError(f"k must have shape {(B, 'H_kv', N, D)}, got {tuple(k.shape)}")
    for x, out, n in ((q, outs[0], "q_out"), (k, outs[1], "k_out")):
        if out is not None and (x is None or out.shape != x.shape):
            raise RuntimeError(f"{n} must have the shape of what is rotated into it")
    _check_rotary(rotary, q.device, D)
    if isinstance(positions, torch.Tensor):
        if positions.dtype not in _INTS or tuple(positions.shape) not in ((N,), (B, N), (1, N)):
            raise RuntimeError(f"positions must be int32 or int64 of shape ({N},) or ({B}, {N}), got {positions.dtype} "
                               f"{tuple(positions.shape)}")
        if positions.device != q.device:
            raise RuntimeError(f"positions must be on {q.device}, got {positions.device}")
    elif not isinstance(positions, int):
        raise RuntimeError(f"positions must be a tensor or the first position, got {type(positions).__name__}")
    elif not _is_first(int(positions)):
        raise RuntimeError(f"the first position must be an integer of 64 bits, got {positions}")


def _rotate(q, k, positions, rotary, q_out, k_out, transposed: bool) -> None:
    """Launches the rotation of what _check_rotate takes."""
    B, H, N, D = q.shape
    if isinstance(positions, torch.Tensor):
        strides = positions.stride()
        # (A single row of positions is every sequence's.)
        strides = (0, strides[-1]) if len(strides) == 1 or positions.shape[0] == 1 else strides
        where, size, first = positions.data_ptr(), positions.element_size(), 0
    else:
        where, size, strides, first = 0, 4, (0, 0), int(positions)
    _launch_on(q.get_device(), _C.rotate, _view(q), _view(q_out), H, _view(k), _view(k_out), 0 if k is None else k.shape[1],
               where, size, strides, first, rotary._turns.data_ptr(), rotary.dim, rotary.interleaved, rotary.magnitude,
               transposed, B, N, D, _ROTATED[q.dtype])


def _empty_like(x):
    """A new tensor in the layout of ``x``, with a dense last dimension: torch's empty_like sorts strides, and puts another
    dimension there where ``x``'s rows share elements (a window that slides by one)."""
    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 or y.shape[-1] <= 1 else x.new_empty(x.shape)


def _dense(x):
    """A gradient as the kernel takes it: an expanded last dimension, for one, is copied."""
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _new_rotated(q, k, positions, rotary, transposed: bool):
    q_out, k_out = _empty_like(q), None if k is None else _empty_like(k)
    _rotate(q, k, positions, rotary, q_out, k_out, transposed)
    return q_out, k_out


def _keep(ctx, positions, rotary, transposed) -> None:
    ctx.rotary, ctx.transposed, ctx.first = rotary, transposed, None
    if isinstance(positions, torch.Tensor):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
    else:
        ctx.first = positions
    # (Forward mode needs a tangent for every result.)
    ctx.set_materialize_grads(getattr(forward_ad, "_current_level", -1) >= 0)


def _again(ctx, q, k, transposed: bool):
    """Tangents or gradients of q and k (one of them may be None), rotated."""
    positions = ctx.saved_tensors[0] if ctx.first is None else ctx.first
    if q is None:
        return None, None if k is None else _differentiable(_dense(k), None, positions, ctx.rotary, transposed)[0]
    return _differentiable(_dense(q), None if k is None else _dense(k), positions, ctx.rotary, transposed)


class _Linear(torch.autograd.Function):
    """The rotation is linear in q and k; its gradient is the transposed rotation."""

    @staticmethod
    def backward(ctx, q, k):
        q, k = _again(ctx, q if ctx.needs_input_grad[0] else None, k if ctx.needs_input_grad[1] else None,
                      not ctx.transposed)
        return q, k, None, None, None

    @staticmethod
    def jvp(ctx, q, k, *_):
        return _again(ctx, q, k, ctx.transposed)


class _Rotate(_Linear):
    @staticmethod
    def forward(ctx, q, k, positions, rotary, transposed):
        _keep(ctx, positions, rotary, transposed)
        outs = _new_rotated(q, k, positions, rotary, transposed)
        needed = ctx.needs_input_grad
        if k is not None and needed[0] != needed[1] and getattr(forward_ad, "_current_level", -1) < 0:  # (tangents: both)
            ctx.mark_non_differentiable(outs[1 if needed[0] else 0])
        return outs


class _RotateTransformed(_Linear):
    """For torch.func's transforms, which ask for the context apart (26 of a call's 37 us on the host)."""

    @staticmethod
    def forward(q, k, positions, rotary, transposed):
        return _new_rotated(q, k, positions, rotary, transposed)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _keep(ctx, *inputs[2:])


def _differentiable(q, k, positions, rotary, transposed: bool):
    """(q', k') as new tensors, part of whatever derivative is being taken."""
    if _transform() is not None:
        return _RotateTransformed.apply(q, k, positions, rotary, transposed)
    if getattr(forward_ad, "_current_level", -1) >= 0 or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
        return _Rotate.apply(q, k, positions, rotary, transposed)
    return _new_rotated(q, k, positions, rotary, transposed)


def rotate(q: torch.Tensor, k: torch.Tensor | None, positions, rotary: Rotary, *, q_out: torch.Tensor | None = None,
           k_out: torch.Tensor | None = None):
    """Rotary positions on queries and keys, in one launch.

    ``q``: (B, H, N, D), ``k``: (B, H_kv, N, D) or None; float32, bf16 or fp16 alike, any strides whose last dimension is
    dense (16-byte pieces are moved whole where strides, D and the rotated dims allow it), D up to 128.  ``positions``:
    int32 or int64 of shape (N,) or (B, N), or an int, the first of N positions in a row.  ``rotary``: a
    :class:`Rotary`; dims past ``rotary.dim`` are copied.  Arithmetic is float32 with one rounding.

    Returns (q', k'), or q' for ``k=None``: new tensors, or ``q_out`` and ``k_out``, of which ``q_out`` may be ``q`` and
    ``k_out`` ``k`` (other overlaps are not taken).  Differentiable with respect to q and k, to any order; with outputs
    given it is not, and refuses inputs that need a gradient.  A captured backward pass needs, as torch's own do, that no
    eager graph of the same leaves lives.
    """
    outs = (q_out, k_out)
    if not _accepts_rotate(q, k, positions, rotary, outs):
        _check_rotate(q, k, positions, rotary, outs)
    if q_out is None and k_out is None:
        q_out, k_out = _differentiable(q, k, positions, rotary, False)
        return q_out if k is None else (q_out, k_out)
    if (_transform() is not None or getattr(forward_ad, "_current_level", -1) >= 0
            or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)))):
        raise RuntimeError("q_out and k_out are not differentiable: rotate without them, or under torch.no_grad()")
    _check_written(q_out, k_out)
    if q_out is None:
        q_out = _empty_like(q)
    if k is not None and k_out is None:
        k_out = _empty_like(k)
    _rotate(q, k, positions, rotary, q_out, k_out, False)
    increment_version([x for x in outs if x is not None])
    return q_out if k is None else (q_out, k_out)


def _are_rows(x, B: int, H: int, N: int, D: int, dtype, index: int) -> bool:
    return x.shape == (B, H, N, D) and x.dtype is dtype and x.get_device() == index and x.stride(3) == 1


def _check_rows(x, name: str, B: int, H: int, N: int, D: int, dtype, dev) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if x.dtype != dtype:
        raise RuntimeError(f"{name} must have dtype {dtype}, got {x.dtype}")
    if tuple(x.shape) != (B, H, N, D):
        raise RuntimeError(f"{name} must have shape {(B, H, N, D)}, got {tuple(x.shape)}")
    if x.device != dev:
        raise RuntimeError(f"{name} must be on {dev}, got {x.device}")
    if x.stride(3) != 1:
        raise RuntimeError(f"{name} must be dense in its last dimension (stride 1), got strides {x.stride()}")


def _check_counts(t, name: str, B: int, dev) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != (B,) or t.device != dev or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous int32 tensor of shape ({B},) on {dev}")


def _accepts_append(k, v, k_pages, v_pages, page_table, cache_seqlens, lengths, rotary, positions, q, q_out) -> bool:
    """Everything _check_append checks, as one test."""
    index, ks = k_pages.get_device(), k.shape
    if not (_accepts_pages(k_pages, v_pages, index) and len(ks) == 4):
        return False
    _, H_kv, _, D = k_pages.shape
    B, N, dtype = ks[0], ks[2], k_pages.dtype
    if not (_are_rows(k, B, H_kv, N, D, dtype, index) and _are_rows(v, B, H_kv, N, D, dtype, index)
            and _is_table(page_table, B, index) and _is_seqlens(cache_seqlens, B, index)):
        return False
    if rotary is None:
        if q is not None or positions is not None:
            return False
    elif not _is_rotary(rotary, index, D):
        return False
    for x in (lengths, positions):
        if x is not None and not _is_seqlens(x, B, index):
            return False
    if q is None:
        return q_out is None
    qs = q.shape
    if len(qs) != 4:
        return False
    return all(x is None or _are_rows(x, B, qs[1], N, D, dtype, index) for x in (q, q_out))


def _check_append(k, v, k_pages, v_pages, page_table, cache_seqlens, lengths, rotary, positions, q, q_out) -> None:
    _check_pages(k_pages, v_pages)
    _, H_kv, _, D = k_pages.shape
    dev, dtype = k_pages.device, k_pages.dtype
    if k.dim() != 4:
        raise RuntimeError(f"k must be 4-D (batch, heads, seq_len, head_dim), got shape {tuple(k.shape)}")
    B, _, N, _ = k.shape
    _check_rows(k, "k", B, H_kv, N, D, dtype, dev)
    _check_rows(v, "v", B, H_kv, N, D, dtype, dev)
    _check_table(page_table, "page_table", B, dev)
    _check_seqlens(cache_seqlens, B, dev)
    if lengths is not None:
        _check_counts(lengths, "lengths", B, dev)
    if rotary is None:
        for x, n in ((q, "q"), (positions, "positions")):
            if x is not None:
                raise RuntimeError(f"{n} needs a rotary")
    else:
        _check_rotary(rotary, dev, D)
    if positions is not None:
        _check_counts(positions, "positions", B, dev)
    if q is None:
        if q_out is not None:
            raise RuntimeError("q_out needs q")
    else:
        if q.dim() != 4:
            raise RuntimeError(f"q must be 4-D (batch, heads, seq_len, head_dim), got shape {tuple(q.shape)}")
        _check_rows(q, "q", B, q.shape[1], N, D, dtype, dev)
        if q_out is not None:
            _check_rows(q_out, "q_out", B, q.shape[1], N, D, dtype, dev)


def append_paged(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, cache_seqlens: torch.Tensor, *, lengths: torch.Tensor | None = None,
                 rotary: Rotary | None = None, positions: torch.Tensor | None = None, q: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None):
    """New tokens' keys and values into a paged cache (:func:`decode_paged`), rotated on the way, in one launch.

    ``k``, ``v``: (B, H_kv, N, D) of the pools' type, any strides as for :func:`attention`.  Token i of sequence b becomes
    its row ``cache_seqlens[b] + i``; with ``lengths`` (int32 (B,)) only the first ``lengths[b]`` of its N tokens do.
    The rows' pages must be the sequence's own, in pools that hold each row in a place of its own; the caller advances
    ``cache_seqlens`` afterwards (after :func:`attend_paged`, which counts the rows before the new tokens too).
    With ``rotary`` the keys are rotated, token i at position ``positions[b] + i`` (int32 (B,); ``cache_seqlens[b] + i``
    without), and so are the queries ``q`` (B, H, N, D), if given: they are returned, in ``q_out`` if given (``q`` itself is
    taken).  Rows of tokens past ``lengths[b]`` are left as they were in ``q_out``, and zeros in a new tensor.

    A sequence whose length or number of new tokens does not fit its table gets no row, and NaN for its queries; a row
    whose page id is outside the pool is not written (checked on the device).
    """
    if not _accepts_append(k, v, k_pages, v_pages, page_table, cache_seqlens, lengths, rotary, positions, q, q_out):
        _check_append(k, v, k_pages, v_pages, page_table, cache_seqlens, lengths, rotary, positions, q, q_out)
    _check_written(k_pages, v_pages, q_out)
    P, H_kv, page, D = k_pages.shape
    B, _, N, _ = k.shape
    pad = q_out is None
    if q is not None and pad:
        q_out = _empty_like(q)
    turns, rot, interleaved, magnitude = (0, 0, False, 1.0) if rotary is None else (
        rotary._turns.data_ptr(), rotary.dim, rotary.interleaved, rotary.magnitude)
    _launch_on(k_pages.get_device(), _C.append, _view(k), _view(v), _view(k_pages), _view(v_pages), page_table.data_ptr(),
               page_table.stride(0), cache_seqlens.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
               0 if positions is None else positions.data_ptr(), _view(q), _view(q_out), pad, turns, rot, interleaved,
               magnitude, B, 0 if q is None else q.shape[1], H_kv, N, P, page, page_table.shape[1], D, _DTYPES[k.dtype])
    increment_version((k_pages, v_pages) if q is None or pad else (k_pages, v_pages, q_out))
    return q_out


def _accepts_attend(q, k_pages, v_pages, page_table, cache_seqlens, lengths, out) -> bool:
    """Everything _check_attend checks, as one test."""
    index, qs = k_pages.get_device(), q.shape
    if not (_accepts_pages(k_pages, v_pages, index) and len(qs) == 4):
        return False
    _, H_kv, _, D = k_pages.shape
    B, H, N, _ = qs
    return (H_kv > 0 and H % H_kv == 0 and _are_rows(q, B, H, N, D, k_pages.dtype, index)
            and (out is None or _are_rows(out, B, H, N, D, k_pages.dtype, index)) and _is_table(page_table, B, index)
            and _is_seqlens(cache_seqlens, B, index) and (lengths is None or _is_seqlens(lengths, B, index)))


def _check_attend(q, k_pages, v_pages, page_table, cache_seqlens, lengths, out) -> None:
    _check_pages(k_pages, v_pages)
    _, H_kv, _, D = k_pages.shape
    dev, dtype = k_pages.device, k_pages.dtype
    if q.dim() != 4:
        raise RuntimeError(f"q must be 4-D (batch, heads, seq_len, head_dim), got shape {tuple(q.shape)}")
    B, H, N, _ = q.shape
    if H_kv == 0 or H % H_kv:
        raise RuntimeError(f"q's {H} heads must be a multiple of the cache's {H_kv}")
    _check_rows(q, "q", B, H, N, D, dtype, dev)
    if out is not None:
        _check_rows(out, "out", B, H, N, D, dtype, dev)
    _check_table(page_table, "page_table", B, dev)
    _check_seqlens(cache_seqlens, B, dev)
    if lengths is not None:
        _check_counts(lengths, "lengths", B, dev)


def attend_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 cache_seqlens: torch.Tensor, *, lengths: torch.Tensor | None = None, causal: bool = True,
                 out: torch.Tensor | None = None, softmax_scale: float | None = None, return_lse: bool = False,
                 workspace: torch.Tensor | None = None):
    """Attention of several new tokens over a paged cache (:func:`decode_paged`) that holds their keys already
    (:func:`append_paged`): a chunk of a prompt, or drafted tokens that are checked together.

    ``q``: (B, H, N, D), any strides as for :func:`attention`, H a multiple of the cache's H_kv.  With ``causal`` token i of
    sequence b sees the ``cache_seqlens[b]`` rows before the new tokens and the new tokens' up to its own; without, every
    token sees the ``cache_seqlens[b]`` rows, all there are (cross attention to cached states of another length).  With
    ``lengths`` (int32 (B,)) only the first ``lengths[b]`` tokens count; rows of the others are left as they were in
    ``out``, and in a new tensor are zeros.  The caller advances ``cache_seqlens`` afterwards.

    Returns ``out`` ((B, H, N, D), new if not given), or ``(out, lse)`` with ``return_lse=True`` (lse (B, H, N) float32,
    natural log, -inf for tokens that do not count).  A token that sees no row, or scores of -inf alone, has output 0 and
    lse -inf.  A sequence whose length or number of new tokens does not fit its table yields NaN for its tokens, a page id
    outside the pool for those that see its rows (checked on the device).  ``workspace`` as for :func:`decode`, of
    ``_C.attend_workspace(B, H, H_kv, N, page, M, D)`` bytes; with a smaller one a tile of rows is one workgroup's.  Keys are
    divided by the table's width: give the columns that the texts may use (a view of a table's first ones).
    """
    if not _accepts_attend(q, k_pages, v_pages, page_table, cache_seqlens, lengths, out):
        _check_attend(q, k_pages, v_pages, page_table, cache_seqlens, lengths, out)
    _check_written(out)
    P, H_kv, page, D = k_pages.shape
    B, H, N, _ = q.shape
    M, index = page_table.shape[1], k_pages.get_device()
    pad = out is None
    if pad:
        out = _empty_like(q)
    lse = None
    if return_lse:
        lse = q.new_empty((B, H, N), dtype=torch.float32)
        if not pad and lengths is not None:
            lse.fill_(-math.inf)  # (with the caller's output the kernel leaves such rows alone)
    scale = (1.0 / math.sqrt(D)) if softmax_scale is None else float(softmax_scale)
    workspace = _workspace(workspace, index, 0 if workspace is not None else
                           _C.attend_workspace(B, H, H_kv, N, page, M, D))
    _launch_on(index, _C.attend, _view(q), _view(k_pages), _view(v_pages), page_table.data_ptr(), page_table.stride(0),
               cache_seqlens.data_ptr(), 0 if lengths is None else lengths.data_ptr(), _view(out),
               0 if lse is None else lse.data_ptr(), pad, bool(causal), B, H, H_kv, N, P, page, M, D, _DTYPES[q.dtype], scale,
               *_extent(workspace))
    if not pad:
        increment_version(out)
    return (out, lse) if return_lse else out


def _accepts_shared(q, k_pages, v_pages, prefix_table, prefix_lens, page_table, cache_seqlens, k_new, v_new, out) -> bool:
    """Everything _check_shared checks, as one test."""
    index, qs = k_pages.get_device(), q.shape
    if not (_accepts_pages(k_pages, v_pages, index) and len(qs) == 3 and (k_new is None) == (v_new is None)
            and len(prefix_table.shape) == 2):
        return False
    _, H_kv, _, D = k_pages.shape
    B, H, _ = qs
    R, dtype = prefix_table.shape[0], k_pages.dtype
    if H_kv == 0 or H % H_kv or R == 0 or B % R:
        return False
    for x, h in ((q, H), (out, H), (k_new, H_kv), (v_new, H_kv)):
        if x is not None and not (x.shape == (B, h, D) and x.dtype is dtype and x.get_device() == index and x.stride(2) == 1):
            return False
    return (_is_table(prefix_table, R, index) and _is_seqlens(prefix_lens, R, index) and _is_table(page_table, B, index)
            and _is_seqlens(cache_seqlens, B, index))


def _check_shared(q, k_pages, v_pages, prefix_table, prefix_lens, page_table, cache_seqlens, k_new, v_new, out) -> None:
    _check_pages(k_pages, v_pages)
    _, H_kv, _, D = k_pages.shape
    dev, dtype = k_pages.device, k_pages.dtype
    if q.dim() != 3:
        raise RuntimeError(f"q must be (B, H, D), got {tuple(q.shape)}")
    B, H, _ = q.shape
    if H_kv == 0 or H % H_kv:
        raise RuntimeError(f"q's {H} heads must be a multiple of the cache's {H_kv}")
    _check_vec(q, "q", B, H, D, dtype, dev)
    R = prefix_table.shape[0] if prefix_table.dim() == 2 else 0
    if R == 0 or B % R:
        raise RuntimeError(f"prefix_table must be int32 of shape (R, pages) with {B} sequences a multiple of R, got "
                           f"{prefix_table.dtype} {tuple(prefix_table.shape)}")
    _check_table(prefix_table, "prefix_table", R, dev)
    _check_counts(prefix_lens, "prefix_lens", R, dev)
    _check_table(page_table, "page_table", B, dev)
    _check_seqlens(cache_seqlens, B, dev)
    if (k_new is None) != (v_new is None):
        raise RuntimeError("k_new and v_new must be given together")
    if k_new is not None:
        _check_vec(k_new, "k_new", B, H_kv, D, dtype, dev)
        _check_vec(v_new, "v_new", B, H_kv, D, dtype, dev)
    if out is not None:
        _check_vec(out, "out", B, H, D, dtype, dev)


def decode_shared(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, prefix_table: torch.Tensor,
                  prefix_lens: torch.Tensor, page_table: torch.Tensor, cache_seqlens: torch.Tensor,
                  k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None, *,
                  out: torch.Tensor | None = None, softmax_scale: float | None = None, return_lse: bool = False,
                  workspace: torch.Tensor | None = None):
    """:func:`decode_paged` for sequences that share their first rows, which are read once for all of them.

    The B sequences of ``q`` (B, H, D) are R groups of B / R, one after the other: sequence b attends to the
    ``prefix_lens[r]`` rows (int32 (R,)) that ``prefix_table`` (int32 (R, M_prefix)) names for its group r = b // (B / R),
    then to the ``cache_seqlens[b]`` rows of its own in ``page_table`` (int32 (B, M)); neither needs to fill its last page.
    Everything else is as for :func:`decode_paged`: the pools, head layouts and types, ``k_new``/``v_new`` ((B, H_kv, D)),
    which become row ``cache_seqlens[b]`` of the sequence's own, ``out``, the lse.  A length that does not fit its table or a
    page id outside the pool yields NaN for the sequence, or for the whole group if it is the prefix's (checked on the
    device).  A prefix's weights are rounded to the type for the product with V, as :func:`attention`'s are, where a group
    has more than 64 query rows (B / R * H / H_kv).  ``workspace``: at least ``_C.decode_shared_workspace(R, B, H, H_kv, page,
    M_prefix, M, D)`` bytes, kept per device and stream where none is given.  Keys are divided by the tables' widths, as in
    :func:`attend_paged`.
    """
    if not _accepts_shared(q, k_pages, v_pages, prefix_table, prefix_lens, page_table, cache_seqlens, k_new, v_new, out):
        _check_shared(q, k_pages, v_pages, prefix_table, prefix_lens, page_table, cache_seqlens, k_new, v_new, out)
    P, H_kv, page, D = k_pages.shape
    B, H, _ = q.shape
    (R, M_prefix), M, index = prefix_table.shape, page_table.shape[1], k_pages.get_device()
    written = ([] if k_new is None else [k_pages, v_pages]) + ([] if out is None else [out])
    _check_written(*written)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, H, D))
    lse = q.new_empty((B, H), dtype=torch.float32) if return_lse else None
    scale = (1.0 / math.sqrt(D)) if softmax_scale is None else float(softmax_scale)
    workspace = _workspace(workspace, index, 0 if workspace is not None else
                           _C.decode_shared_workspace(R, B, H, H_kv, page, M_prefix, M, D))
    _launch_on(index, _C.decode_shared, _view(q), _view(k_pages), _view(v_pages), prefix_table.data_ptr(),
               prefix_table.stride(0), prefix_lens.data_ptr(), page_table.data_ptr(), page_table.stride(0),
               cache_seqlens.data_ptr(), _NONE3 if k_new is None else _view(k_new), _NONE3 if v_new is None else _view(v_new),
               _view(out), 0 if lse is None else lse.data_ptr(), R, B, H, H_kv, P, page, M_prefix, M, D, _DTYPES[q.dtype],
               scale, *_extent(workspace))
    if written:
        increment_version(written)
    return (out, lse) if return_lse else out
