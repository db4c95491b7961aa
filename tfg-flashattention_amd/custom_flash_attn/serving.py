"""The serving operators beside the attention (include/tfgfa_serving.h) on torch tensors: a decode step
over a paged KV cache, the attention weight each key receives, eviction from the cache by that weight,
and penalties, biases and grammar masks on logits.

The reference's generate() has no cache and samples from unmodified logits
(src/py/model_inference.py:199-228); nothing here has a counterpart in it.  The functions check their
arguments (RuntimeError, before anything is launched), launch on the current stream of the tensors'
device and do not synchronise.
"""
from __future__ import annotations

import math

import torch

from . import _C, _DTYPES, MAX_HEAD_DIM, _check_vec, _current_stream, _decode_workspace, _launch_on, _WORKSPACES

_ZERO2, _ZERO3 = (0, 0), (0, 0, 0)
_LOGITS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check_pages(k_pages, v_pages) -> None:
    for t, n in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not t.is_cuda:
            raise RuntimeError(f"{n} must be a CUDA tensor")
        if t.dtype not in _DTYPES:
            raise RuntimeError("Unsupported tensor dtype. Use bfloat16 or float16.")
        if t.dim() != 4:
            raise RuntimeError(f"{n} must be (P, H_kv, page, D), got {tuple(t.shape)}")
        if t.stride(3) != 1:
            raise RuntimeError(f"{n} must be dense in its last dimension (stride 1), got strides {t.stride()}")
    if not (8 <= k_pages.shape[3] <= MAX_HEAD_DIM and k_pages.shape[3] % 8 == 0):
        raise RuntimeError(f"head_dim must be a multiple of 8 in [8, {MAX_HEAD_DIM}], got {k_pages.shape[3]}")
    if k_pages.shape[2] < 1:
        raise RuntimeError("a page holds at least one row")
    if v_pages.dtype != k_pages.dtype:
        raise RuntimeError(f"v_pages must have dtype {k_pages.dtype}, got {v_pages.dtype}")
    if v_pages.shape != k_pages.shape:
        raise RuntimeError(f"v_pages must have shape {tuple(k_pages.shape)}, got {tuple(v_pages.shape)}")
    if v_pages.device != k_pages.device:
        raise RuntimeError(f"v_pages must be on {k_pages.device}, got {v_pages.device}")


def _check_table(t, name: str, B: int, dev) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != B:
        raise RuntimeError(f"{name} must be int32 of shape ({B}, pages)")
    if t.device != dev or (t.shape[1] > 1 and t.stride(1) != 1):
        raise RuntimeError(f"{name} must be on {dev} and dense in its last dimension")


def _check_seqlens(t, B: int, dev) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != (B,):
        raise RuntimeError(f"cache_seqlens must be int32 of shape ({B},)")
    if t.device != dev or not t.is_contiguous():
        raise RuntimeError(f"cache_seqlens must be a contiguous tensor on {dev}")


def _check_weights(t, name: str, B: int, H_kv: int, rows: int, dev) -> None:
    if t.dtype != torch.float32 or t.dim() != 3 or tuple(t.shape[:2]) != (B, H_kv) or t.shape[2] < rows:
        raise RuntimeError(f"{name} must be float32 of shape ({B}, {H_kv}, at least {rows}), got {t.dtype} "
                           f"{tuple(t.shape)}")
    if t.device != dev or (t.shape[2] > 1 and t.stride(2) != 1):
        raise RuntimeError(f"{name} must be on {dev} and dense in its last dimension")


def _workspace(given, index: int, nbytes: int):
    """The caller's workspace, checked, or one of at least ``nbytes`` for device ``index``'s current stream; None where
    none is needed.  The caller keeps it until after the launch: another thread's call on the stream may replace the
    kept one by a larger one in between, and its memory would go to the next tensor."""
    if given is not None:
        if not given.is_cuda or given.get_device() != index or not given.is_contiguous():
            raise RuntimeError(f"workspace must be a contiguous tensor on cuda:{index}")
        return given
    if not nbytes:
        return None
    dev = torch.device("cuda", index)
    workspace = None if torch.cuda.is_current_stream_capturing() else _WORKSPACES.get((dev, _current_stream(index)))
    if workspace is None or workspace.numel() < nbytes:
        workspace = _decode_workspace(dev, nbytes)
    return workspace


def _extent(workspace) -> tuple[int, int]:
    """(pointer, bytes) of a workspace or None."""
    return (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())


def _accepts_pages(k_pages, v_pages, index) -> bool:
    """Everything _check_pages checks, as one test."""
    ks, dtype = k_pages.shape, k_pages.dtype
    return (index >= 0 and k_pages.is_cuda and dtype in _DTYPES and len(ks) == 4 and v_pages.shape == ks
            and v_pages.dtype is dtype and v_pages.get_device() == index and ks[2] >= 1
            and 8 <= ks[3] <= MAX_HEAD_DIM and ks[3] % 8 == 0 and k_pages.stride(3) == 1 and v_pages.stride(3) == 1)


def _is_table(t, B: int, index: int) -> bool:
    s = t.shape
    return (t.dtype is torch.int32 and len(s) == 2 and s[0] == B and t.get_device() == index
            and (s[1] <= 1 or t.stride(1) == 1))


def _is_seqlens(t, B: int, index: int) -> bool:
    return t.dtype is torch.int32 and t.shape == (B,) and t.get_device() == index and t.is_contiguous()


def _are_weights(t, B: int, H_kv: int, rows: int, index: int) -> bool:
    s = t.shape
    return (t.dtype is torch.float32 and len(s) == 3 and s[0] == B and s[1] == H_kv and s[2] >= rows
            and t.get_device() == index and (s[2] <= 1 or t.stride(2) == 1))


def _accepts_paged(q, k_pages, v_pages, page_table, cache_seqlens, k_new, v_new, key_weights, out) -> bool:
    """Everything _check_paged checks, as one test."""
    index, qs = k_pages.get_device(), q.shape
    if not (_accepts_pages(k_pages, v_pages, index) and len(qs) == 3 and (k_new is None) == (v_new is None)):
        return False
    _, H_kv, page, D = k_pages.shape
    B, H, _ = qs
    if H_kv == 0 or H % H_kv or not (_is_table(page_table, B, index) and _is_seqlens(cache_seqlens, B, index)):
        return False
    dtype = k_pages.dtype
    for x, h in ((q, H), (out, H), (k_new, H_kv), (v_new, H_kv)):
        if x is not None and not (x.shape == (B, h, D) and x.dtype is dtype and x.get_device() == index
                                  and x.stride(2) == 1):
            return False
    return key_weights is None or _are_weights(key_weights, B, H_kv, page_table.shape[1] * page, index)


def _check_paged(q, k_pages, v_pages, page_table, cache_seqlens, k_new, v_new, key_weights, out) -> None:
    _check_pages(k_pages, v_pages)
    _, H_kv, page, D = k_pages.shape
    dev, dtype = k_pages.device, k_pages.dtype
    if q.dim() != 3:
        raise RuntimeError(f"q must be (B, H, D), got {tuple(q.shape)}")
    B, H, _ = q.shape
    if H_kv == 0 or H % H_kv:
        raise RuntimeError(f"q's {H} heads must be a multiple of the cache's {H_kv}")
    _check_vec(q, "q", B, H, D, dtype, dev)
    _check_table(page_table, "page_table", B, dev)
    _check_seqlens(cache_seqlens, B, dev)
    if (k_new is None) != (v_new is None):
        raise RuntimeError("k_new and v_new must be given together")
    if k_new is not None:
        _check_vec(k_new, "k_new", B, H_kv, D, dtype, dev)
        _check_vec(v_new, "v_new", B, H_kv, D, dtype, dev)
    if out is not None:
        _check_vec(out, "out", B, H, D, dtype, dev)
    if key_weights is not None:
        _check_weights(key_weights, "key_weights", B, H_kv, page_table.shape[1] * page, dev)


def decode_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 cache_seqlens: torch.Tensor, k_new: torch.Tensor | None = None,
                 v_new: torch.Tensor | None = None, *, key_weights: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, softmax_scale: float | None = None, return_lse: bool = False,
                 workspace: torch.Tensor | None = None):
    """:func:`decode` over a paged cache, with query heads that may share key-value heads.

    ``q``: (B, H, D).  ``k_pages``, ``v_pages``: (P, H_kv, page, D) pools (any strides with a dense last
    dimension, e.g. (P, page, H_kv, D) buffers transposed); H a multiple of H_kv, query head h reading
    key-value head ``h // (H // H_kv)``; any page size.  bf16 or fp16, all alike; D a multiple of 8 up to
    128.  ``page_table``: int32 (B, M); row j of sequence b is row ``j % page`` of page
    ``page_table[b, j // page]``.  ``cache_seqlens``: int32 (B,), the cached rows; entries of the table
    past them are not used.  With ``k_new``/``v_new`` ((B, H_kv, D)) the new token becomes row
    ``cache_seqlens[b]`` first (its page must be the sequence's own) and is attended too; the caller
    advances ``cache_seqlens`` afterwards.  Pages may otherwise be shared by sequences.  Pools that are appended to
    hold each row in a place of its own (no expanded views).  bf16 values past 3.4e38 / (2981 rows) can make float32's
    sums infinite.

    ``key_weights``: float32 (B, H_kv, N >= M * page), the attention weight each row has received: this
    step's softmax weights, summed over the query heads of each key-value head, are added in place (for
    a new row: set).  A head whose log-sum-exp is not finite adds nothing.

    Returns ``out`` ((B, H, D), new if not given), or ``(out, lse)`` with ``return_lse=True`` (lse (B, H)
    float32, natural log).  A length that does not fit its table, or a page id outside the pool among a
    sequence's rows, yields NaN for that batch row (checked on the device).  ``workspace`` as for
    :func:`decode`, of ``_C.decode_paged_workspace(B, H, H_kv, page, M, D, with_weights)`` bytes; a smaller
    one is refused with ``key_weights`` and otherwise runs each key-value head as one workgroup.
    """
    if not _accepts_paged(q, k_pages, v_pages, page_table, cache_seqlens, k_new, v_new, key_weights, out):
        _check_paged(q, k_pages, v_pages, page_table, cache_seqlens, k_new, v_new, key_weights, out)
    P, H_kv, page, D = k_pages.shape
    B, H, _ = q.shape
    M, index = page_table.shape[1], k_pages.get_device()
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, H, D))
    scale = (1.0 / math.sqrt(D)) if softmax_scale is None else float(softmax_scale)
    lse = q.new_empty((B, H), dtype=torch.float32) if return_lse else None
    workspace = _workspace(workspace, index, 0 if workspace is not None else
                           _C.decode_paged_workspace(B, H, H_kv, page, M, D, key_weights is not None))
    _launch_on(index, _C.decode_paged,
               q.data_ptr(), q.stride(), k_pages.data_ptr(), k_pages.stride(), v_pages.data_ptr(), v_pages.stride(),
               page_table.data_ptr(), page_table.stride(0), cache_seqlens.data_ptr(),
               0 if k_new is None else k_new.data_ptr(), _ZERO3 if k_new is None else k_new.stride(),
               0 if v_new is None else v_new.data_ptr(), _ZERO3 if v_new is None else v_new.stride(),
               out.data_ptr(), out.stride(), 0 if lse is None else lse.data_ptr(),
               0 if key_weights is None else key_weights.data_ptr(),
               _ZERO2 if key_weights is None else key_weights.stride()[:2],
               B, H, H_kv, P, page, M, D, _DTYPES[q.dtype], scale, *_extent(workspace))
    return (out, lse) if return_lse else out


def _accepts_weights(q, k, lse, first_query, out) -> bool:
    """Everything _check_key_weights checks, as one test."""
    qs, ks, dtype, index = q.shape, k.shape, q.dtype, q.get_device()
    if not (index >= 0 and q.is_cuda and dtype in _DTYPES and k.dtype is dtype and k.get_device() == index
            and len(qs) == 4 and len(ks) == 4 and ks[0] == qs[0] and ks[3] == qs[3]
            and 8 <= qs[3] <= MAX_HEAD_DIM and qs[3] % 8 == 0 and q.stride(3) == 1 and k.stride(3) == 1
            and ks[1] and qs[1] and qs[1] % ks[1] == 0 and first_query >= 0):
        return False
    return (lse.dtype is torch.float32 and lse.shape == qs[:3] and lse.get_device() == index
            and (qs[2] <= 1 or lse.stride(2) == 1)
            and (out is None or (out.shape == ks[:3] and _are_weights(out, ks[0], ks[1], ks[2], index))))


def _check_key_weights(q, k, lse, first_query, out) -> None:
    for t, n in ((q, "q"), (k, "k")):
        if not t.is_cuda:
            raise RuntimeError(f"{n} must be a CUDA tensor")
        if t.dtype not in _DTYPES:
            raise RuntimeError("Unsupported tensor dtype. Use bfloat16 or float16.")
        if t.dim() != 4:
            raise RuntimeError(f"{n} must be 4-D (batch, heads, seq_len, head_dim), got shape {tuple(t.shape)}")
        if t.stride(3) != 1:
            raise RuntimeError(f"{n} must be dense in its last dimension (stride 1), got strides {t.stride()}")
    B, H, N_q, D = q.shape
    H_kv, N_k, dev = k.shape[1], k.shape[2], q.device
    if k.dtype != q.dtype:
        raise RuntimeError(f"k must have dtype {q.dtype}, got {k.dtype}")
    if k.device != dev:
        raise RuntimeError(f"k must be on {dev}, got {k.device}")
    if k.shape[0] != B or k.shape[3] != D:
        raise RuntimeError(f"k must have shape {(B, 'H_kv', 'N_k', D)}, got {tuple(k.shape)}")
    if not (8 <= D <= MAX_HEAD_DIM and D % 8 == 0):
        raise RuntimeError(f"head_dim must be a multiple of 8 in [8, {MAX_HEAD_DIM}], got {D}")
    if H_kv == 0 or H == 0 or H % H_kv:
        raise RuntimeError(f"q's {H} heads must be a multiple of k's {H_kv}")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, N_q):
        raise RuntimeError(f"lse must be float32 of shape {(B, H, N_q)}, got {lse.dtype} {tuple(lse.shape)}")
    if lse.device != dev or (N_q > 1 and lse.stride(2) != 1):
        raise RuntimeError(f"lse must be on {dev} and dense in its last dimension")
    if first_query < 0:
        raise RuntimeError(f"first_query must not be negative, got {first_query}")
    if out is not None:
        _check_weights(out, "out", B, H_kv, N_k, dev)
        if out.shape[2] != N_k:
            raise RuntimeError(f"out must have shape {(B, H_kv, N_k)}, got {tuple(out.shape)}")


def key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, *, first_query: int = 0,
                out: torch.Tensor | None = None, softmax_scale: float | None = None, causal: bool = True,
                workspace: torch.Tensor | None = None):
    """The attention weight each key receives from given queries: what a cache's ``key_weights``
    (:func:`decode_paged`) start from after a prompt.

    ``out[b, h', j]`` is the sum, over the query heads h of key-value head h' and the queries i that see key
    j, of ``exp(scale * q[b,h,i] . k[b,h',j] - lse[b,h,i])``.  ``q``: (B, H, N_q, D), ``k``: (B, H_kv, N_k,
    D), bf16 or fp16 views as for :func:`attention`, D a multiple of 8 up to 128, H a multiple of H_kv.
    ``lse``: float32 (B, H, N_q) with a dense last dimension, as :func:`attention` returned it for these
    queries.  Query i stands at position ``first_query + i`` and with ``causal`` sees the keys up to it: the
    last w queries of a prompt of N are ``q[:, :, -w:]``, ``lse[:, :, -w:]`` with ``first_query=N - w``.
    A query whose lse is -inf adds nothing.  Returns ``out``, float32 (B, H_kv, N_k) (new if not given; a view
    into a cache's weights with a dense last dimension is taken).  Sums are added in a fixed order.
    ``workspace`` as for :func:`decode`, of ``_C.key_weights_workspace(B, H, H_kv, N_q, N_k, causal)`` bytes (0 where
    the keys fill the device); with a smaller one a block of keys is one workgroup's, whatever its queries.
    """
    if not _accepts_weights(q, k, lse, first_query, out):
        _check_key_weights(q, k, lse, first_query, out)
    B, H, N_q, D = q.shape
    H_kv, N_k = k.shape[1], k.shape[2]
    if out is None:
        out = lse.new_empty((B, H_kv, N_k))
    scale = (1.0 / math.sqrt(D)) if softmax_scale is None else float(softmax_scale)
    index = q.get_device()
    workspace = _workspace(workspace, index, 0 if workspace is not None else
                           _C.key_weights_workspace(B, H, H_kv, N_q, N_k, bool(causal)))
    _launch_on(index, _C.key_weights, q.data_ptr(), q.stride(), k.data_ptr(), k.stride(),
               lse.data_ptr(), lse.stride()[:2], out.data_ptr(), out.stride()[:2], B, H, H_kv, N_q, N_k, D,
               _DTYPES[q.dtype], scale, bool(causal), first_query, *_extent(workspace))
    return out


def _check_evict(k_pages, v_pages, page_table, cache_seqlens, key_weights, new_page_table, budget, recent,
                 weights_out, B) -> None:
    _check_pages(k_pages, v_pages)
    _, H_kv, page, _ = k_pages.shape
    dev = k_pages.device
    _check_seqlens(cache_seqlens, B, dev)
    _check_table(page_table, "page_table", B, dev)
    _check_table(new_page_table, "new_page_table", B, dev)
    _check_weights(key_weights, "key_weights", B, H_kv, page_table.shape[1] * page, dev)
    if not 0 <= recent <= budget:
        raise RuntimeError(f"recent must be between 0 and budget ({budget}), got {recent}")
    if new_page_table.shape[1] * page < budget:
        raise RuntimeError(f"new_page_table's {new_page_table.shape[1]} pages of {page} rows do not hold "
                           f"{budget} rows")
    if weights_out is not None:
        _check_weights(weights_out, "weights_out", B, H_kv, budget, dev)


def evict(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, cache_seqlens: torch.Tensor,
          key_weights: torch.Tensor, new_page_table: torch.Tensor, budget: int, *, recent: int = 0,
          weights_out: torch.Tensor | None = None):
    """Cuts each sequence of a paged cache (:func:`decode_paged`) to ``budget`` rows by attention weight.

    For each sequence and key-value head the last ``recent`` of its rows stay, then those of the largest
    ``key_weights`` (float32 (B, H_kv, N >= M * page)), ties to the lowest row; NaN ranks below every
    number.  The ``n = min(cache_seqlens[b], budget)`` rows kept are copied, in their order, to rows
    0 .. n - 1 of the pages that ``new_page_table`` (int32 (B, M_new), ``M_new * page >= budget``) names;
    entries past row n are not read.  Those pages must be ones that no row still reads, each named once, in pools that
    hold each row in a place of its own.  The old pages are left as they were, so that other sequences may go on
    sharing them.  Afterwards the caller takes ``new_page_table`` for the sequences' and bounds ``cache_seqlens`` by
    ``budget``.

    Returns ``(kept, weights)``: int32 (B, H_kv, budget), the kept rows, -1 from n on, and float32 (B,
    H_kv, budget), their weights, 0 from n on.  With ``weights_out`` (float32 (B, H_kv, at least budget); it
    may be ``key_weights`` itself) the weights are written to its first ``budget`` columns and it is returned
    for them.  A length that does not fit its table, or a page id outside the pool among the ones a
    sequence needs, yields -1 and NaN, and nothing is copied for it (checked on the device).
    """
    index, M_new = k_pages.get_device(), new_page_table.shape[-1]
    B = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else -1
    if not (_accepts_pages(k_pages, v_pages, index) and _is_seqlens(cache_seqlens, B, index)
            and _is_table(page_table, B, index) and _is_table(new_page_table, B, index) and 0 <= recent <= budget
            and M_new * k_pages.shape[2] >= budget
            and _are_weights(key_weights, B, k_pages.shape[1], page_table.shape[1] * k_pages.shape[2], index)
            and (weights_out is None or _are_weights(weights_out, B, k_pages.shape[1], budget, index))):
        _check_evict(k_pages, v_pages, page_table, cache_seqlens, key_weights, new_page_table, budget, recent,
                     weights_out, B)
    P, H_kv, page, D = k_pages.shape
    if weights_out is None:
        weights_out = key_weights.new_empty((B, H_kv, budget))
    kept = cache_seqlens.new_empty((B, H_kv, budget))
    _launch_on(index, _C.evict, k_pages.data_ptr(), k_pages.stride(), v_pages.data_ptr(),
               v_pages.stride(), page_table.data_ptr(), page_table.stride(0), cache_seqlens.data_ptr(),
               key_weights.data_ptr(), key_weights.stride()[:2], new_page_table.data_ptr(), new_page_table.stride(0),
               kept.data_ptr(), weights_out.data_ptr(), weights_out.stride()[:2], B, H_kv, P, page,
               page_table.shape[1], M_new, D, budget, recent)
    return kept, weights_out


def _penalty(p, name: str, B: int, dev):
    """(device pointer or 0, scalar) of a penalty given as a number or as one float32 per row."""
    if not isinstance(p, torch.Tensor):
        p = float(p)
        if not math.isfinite(p) or (name == "repetition" and p <= 0):
            raise RuntimeError(f"{name} must be finite{' and positive' if name == 'repetition' else ''}, got {p}")
        return 0, p
    if p.dtype != torch.float32 or tuple(p.shape) != (B,) or p.device != dev or not p.is_contiguous():
        raise RuntimeError(f"{name} must be a number or a contiguous float32 tensor of shape ({B},) on {dev}")
    return p.data_ptr(), 1.0


def _is_rows(t, dtype, B: int, width: int, index: int) -> bool:
    s = t.shape
    return (t.dtype is dtype and (s == (width,) or s == (B, width)) and t.get_device() == index
            and (width <= 1 or t.stride(-1) == 1))


def _accepts_logits(logits, tokens, lengths, bias, allowed, out) -> bool:
    """Everything _check_logits checks, as one test."""
    s, index = logits.shape, logits.get_device()
    if not (index >= 0 and logits.is_cuda and logits.dtype in _LOGITS and len(s) == 2
            and (s[1] <= 1 or logits.stride(1) == 1)):
        return False
    B, V = s
    if tokens is None:
        if lengths is not None:
            return False
    else:
        ts = tokens.shape
        if not (tokens.dtype in (torch.int64, torch.int32) and len(ts) == 2 and ts[0] == B
                and tokens.get_device() == index and (ts[1] <= 1 or tokens.stride(1) == 1)
                and (lengths is None or _is_seqlens(lengths, B, index))):
            return False
    return ((bias is None or _is_rows(bias, torch.float32, B, V, index))
            and (allowed is None or _is_rows(allowed, torch.int32, B, -(-V // 32), index))
            and (out is None or (out.dtype is logits.dtype and out.shape == s and out.get_device() == index
                                 and (V <= 1 or out.stride(1) == 1))))


def _check_logits(logits, tokens, lengths, bias, allowed, out) -> None:
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA tensor")
    if logits.dtype not in _LOGITS:
        raise RuntimeError("Unsupported tensor dtype. Use float32, bfloat16 or float16.")
    if logits.dim() != 2:
        raise RuntimeError(f"logits must be (B, V), got {tuple(logits.shape)}")
    B, V = logits.shape
    dev = logits.device
    if V > 1 and logits.stride(1) != 1:
        raise RuntimeError(f"logits must be dense in its last dimension (stride 1), got strides {logits.stride()}")
    if tokens is not None:
        if tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() != 2 or tokens.shape[0] != B:
            raise RuntimeError(f"tokens must be int32 or int64 of shape ({B}, T), got {tokens.dtype} "
                               f"{tuple(tokens.shape)}")
        if tokens.device != dev or (tokens.shape[1] > 1 and tokens.stride(1) != 1):
            raise RuntimeError(f"tokens must be on {dev} and dense in its last dimension")
    if lengths is not None:
        if tokens is None:
            raise RuntimeError("lengths needs tokens")
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,) or lengths.device != dev \
                or not lengths.is_contiguous():
            raise RuntimeError(f"lengths must be a contiguous int32 tensor of shape ({B},) on {dev}")
    for t, n, dtype, width in ((bias, "bias", torch.float32, V), (allowed, "allowed", torch.int32, -(-V // 32))):
        if t is not None and (t.dtype != dtype or tuple(t.shape) not in ((width,), (B, width)) or t.device != dev
                              or (width > 1 and t.stride(-1) != 1)):
            raise RuntimeError(f"{n} must be {dtype} of shape ({width},) or ({B}, {width}) on {dev}, dense in its "
                               "last dimension")
    if out is not None and (out.dtype != logits.dtype or out.shape != logits.shape or out.device != dev
                            or (V > 1 and out.stride(1) != 1)):
        raise RuntimeError(f"out must be {logits.dtype} of shape {(B, V)} on {dev}, dense in its last dimension")


def penalize_logits(logits: torch.Tensor, tokens: torch.Tensor | None = None, *,
                    lengths: torch.Tensor | None = None, repetition=1.0, presence=0.0, frequency=0.0,
                    bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                    out: torch.Tensor | None = None):
    """Penalties for repeated tokens, biases and a grammar's mask on logits, in one pass.

    ``logits``: (B, V) float32, bf16 or fp16, last dimension dense.  ``tokens``: int32 or int64 (B, T), the
    text so far, of which row b counts its first ``lengths[b]`` (int32 (B,), taken into [0, T]; all
    without it); ids outside [0, V) count for nothing, so padding may be -1.  A token that stands n > 0
    times in it has its logit x divided (x > 0) or multiplied (x <= 0) by ``repetition``, then lowered by
    ``n * frequency + presence``; each of the three is a number or a float32 (B,) tensor.  ``bias``: float32
    (V,) or (B, V), added to all.  ``allowed``: int32 (ceil(V / 32),) or (B, ceil(V / 32)) words whose bit
    ``v % 32`` of word ``v // 32`` allows token v; the others become -inf whatever they held.
    Arithmetic is float32 with one rounding to the logits' type.  Returns ``out`` (new if not given;
    ``logits`` itself is taken, other overlaps are not).
    """
    if not _accepts_logits(logits, tokens, lengths, bias, allowed, out):
        _check_logits(logits, tokens, lengths, bias, allowed, out)
    B, V = logits.shape
    dev = logits.device
    repetition = _penalty(repetition, "repetition", B, dev)
    presence = _penalty(presence, "presence", B, dev)
    frequency = _penalty(frequency, "frequency", B, dev)
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((B, V))
    T = 0 if tokens is None else tokens.shape[1]
    _launch_on(logits.get_device(), _C.penalize, logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0),
               _LOGITS[logits.dtype], 0 if tokens is None else tokens.data_ptr(),
               8 if tokens is None else tokens.element_size(), 0 if tokens is None else tokens.stride(0),
               0 if lengths is None else lengths.data_ptr(), *repetition, *presence, *frequency,
               0 if bias is None else bias.data_ptr(), 0 if bias is None or bias.dim() == 1 else bias.stride(0),
               0 if allowed is None else allowed.data_ptr(),
               0 if allowed is None or allowed.dim() == 1 else allowed.stride(0), B, V, T)
    return out
