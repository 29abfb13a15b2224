"""Serving from a paged cache: new keys and values into pages, attention over them.

``paged_append`` writes the keys and values of new tokens into the pages of their sequences, rotated by their positions on the
way, and ``paged_attention`` attends to them; both read lengths, rows and pages on the device, so that a captured call serves
later steps as well.  The conventions both share:

* ``k_cache``, ``v_cache``: (pages, page_size, Hkv, D), fp16 or bf16; any strides with the head dimension contiguous, so a
  cache laid out (pages, Hkv, page_size, D) is passed as its ``transpose(1, 2)``.  ``page_size`` is a power of two from 16 to
  1024.
* ``block_table``: (B, columns) int32; token j of sequence b lies in page ``block_table[b, j // page_size]``.  Entries whose
  tokens nobody needs (past a sequence's end, slid out of the window) may hold anything.
* ``seq_lens``: (B,) int32, the tokens of each sequence, the new ones among them and last: new token i of n sits at position
  ``seq_lens[b] - n + i``.  A sequence of length 0 takes no part: its rows of the result are 0.
* New tokens come as (B, n, heads, D), or ragged as (rows, heads, D) with ``cu_q``, (B + 1,) int32: the rows of sequence b are
  ``cu_q[b]`` to ``cu_q[b + 1] - 1``.  Rows before the first sequence's and behind the last one's are left as they are.

A length, row, page or position outside these tensors is found on the device, also in a sequence that has no rows: it sets a bit
that :func:`miniattn.check_device_status` turns into an error, nothing outside them is read or written, and that sequence's
results are undefined.  Row numbers that fall leave those of the whole call undefined, and so does a page outside the cache among
those of a shared prefix.  The tensors must not change while a call runs.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .ops import (_DTYPES, _INT32_MAX, _as_int, _cache_scratch_bytes, _current_device, _current_raw_stream, _launch_cache, _status_word,
                  _status_words)

# What follows from the shapes, strides, dtypes and devices of a call, once they have been checked: the part of the parameter
# block behind the pointers, and the scratch that is needed.  A serving loop passes tensors of the same form step after step.
_attend_forms: dict = {}
_append_forms: dict = {}
_FORMS_MAX = 1024
_pack_attend = struct.Struct("@9P").pack    # the pointers of MiniAttnCacheParams, in one go
_pack_append = struct.Struct("@11P").pack   # and of MiniAttnAppendParams
_ATTEND_POINTERS, _APPEND_POINTERS = 9 * struct.calcsize("P"), 11 * struct.calcsize("P")


def rope_table(positions: int, dim: int, *, theta: float = 10000.0, device: Union[torch.device, str, None] = None) -> torch.Tensor:
    """The rotation table that :func:`paged_append` takes: (positions, dim) fp32, the cosines of the angles
    ``pos * theta**(-2 i / dim)`` of each position, i < dim / 2, and then their sines, taken in 64 bits and rounded once (an
    angle of position 10**6 has lost four digits in 32)."""
    if dim <= 0 or dim % 2:
        raise RuntimeError(f"dim must be positive and even, got {dim}")
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * theta ** (-2.0 * i / dim)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _check(name: str, t, like: Optional[torch.Tensor], dims: int) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if like is not None and t.device != like.device:
        raise RuntimeError("Input tensors must be on the same device")
    if t.dim() != dims:
        raise RuntimeError(f"{name} must be {dims}-D, got {t.dim()}-D")


def _check_half(name: str, t, like: Optional[torch.Tensor], dims: int) -> None:
    _check(name, t, like, dims)
    if t.dtype not in _DTYPES:
        raise RuntimeError("Only fp16 and bf16 are supported")
    if like is not None and t.dtype != like.dtype:
        raise RuntimeError("Input tensors must have the same data type")
    if t.stride(-1) != 1 and t.numel() > 0:
        raise RuntimeError(f"{name} must be contiguous in the head dimension")


def _check_ints(name: str, t, like: torch.Tensor, shape: Tuple[Optional[int], ...]) -> None:
    _check(name, t, like, len(shape))
    if t.dtype != torch.int32:
        raise RuntimeError(f"{name} must be int32")
    if any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise RuntimeError(f"{name} must have the shape {tuple('*' if n is None else n for n in shape)}, got {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise RuntimeError(f"{name} must be contiguous in its last dimension")


def _whole(name: str, x: int, low: int) -> int:
    if x < low or x > _INT32_MAX:
        raise RuntimeError(f"{name} must be between {low} and {_INT32_MAX}, got {x}")
    return x


def _check_paged(new: torch.Tensor, k_cache, v_cache, block_table, seq_lens, cu_q) -> int:
    """Everything but `new` itself, which gives device and dtype; returns the number of sequences."""
    _check_half("k_cache", k_cache, new, 4)
    _check_half("v_cache", v_cache, new, 4)
    if k_cache.shape != v_cache.shape:
        raise RuntimeError("k_cache and v_cache must have the same shape")
    if k_cache.shape[3] != new.shape[-1]:
        raise RuntimeError("the new tokens and the cache must agree in head dim")
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise RuntimeError("block_table must be a 2-D CUDA tensor")
    if max(*new.shape, *k_cache.shape, *block_table.shape) > _INT32_MAX:
        raise RuntimeError("sizes must fit in 31 bits")
    B = block_table.shape[0]
    _check_ints("block_table", block_table, new, (B, None))
    _check_ints("seq_lens", seq_lens, new, (B,))
    if cu_q is not None:
        _check_ints("cu_q", cu_q, new, (B + 1,))
        if new.dim() != 3:
            raise RuntimeError("ragged tokens (cu_q) must be (rows, heads, D)")
    elif new.dim() != 4 or new.shape[0] != B:
        raise RuntimeError(f"new tokens must be ({B}, tokens, heads, D), or (rows, heads, D) with cu_q")
    return B


def _token_strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """(sequence, head, token) of (B, n, heads, D) or (rows, heads, D)"""
    return (t.stride(0), t.stride(2), t.stride(1)) if t.dim() == 4 else (0, t.stride(1), t.stride(0))


def _page_strides(t: torch.Tensor) -> Tuple[int, int, int]:
    return t.stride(0), t.stride(2), t.stride(1)


def _form(t: Optional[torch.Tensor]):
    """What the checks look at."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _keep(forms: dict, key, value):
    if key is not None:
        if len(forms) >= _FORMS_MAX:
            forms.clear()
        forms[key] = value
    return value


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    cu_q: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
    rope: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> Optional[torch.Tensor]:
    """Write the keys and values of new tokens into the pages of their sequences (conventions: module docstring).

    With ``rope`` (a table of :func:`rope_table`, its width the rotated part of each head, a multiple of 16) the keys are
    rotated by their positions on the way, and so is ``q``, the queries of the same tokens, which come back in ``q_out``
    (a new tensor by default; ``q`` itself is fine, any other overlap is not).  Pairs are elements (i, i + width / 2) of a
    head, neighbours (2 i, 2 i + 1) with ``interleaved``.  Tokens at negative positions (the front of a padded sequence,
    ``seq_lens[b] < n``) are left out and their queries copied; so are tokens whose position or page is out of range.  Two
    tokens of one call must not go to the same place of the cache, which a block table that gives a page to one writing
    sequence at a time ensures.

    Returns the rotated queries, or None without ``q``.
    """
    interleaved = bool(interleaved)
    try:
        key = (_form(k), _form(v), _form(k_cache), _form(v_cache), _form(block_table), _form(seq_lens), _form(cu_q), _form(q),
               _form(q_out), _form(rope), interleaved)
        form = _append_forms.get(key)
    except (AttributeError, TypeError, RuntimeError):   # not tensors: let the checks below say so
        key = form = None
    if form is None:
        _check_half("k", k, None, 4 if cu_q is None else 3)
        _check_half("v", v, k, k.dim())
        B = _check_paged(k, k_cache, v_cache, block_table, seq_lens, cu_q)
        if v.shape != k.shape:
            raise RuntimeError("k and v must have the same shape")
        if k.shape[-2] != k_cache.shape[2]:
            raise RuntimeError("k and the cache must agree in heads")
        if k.shape[-2] == 0:
            raise RuntimeError("the number of KV heads must be positive")
        if q is None and q_out is not None:
            raise RuntimeError("q_out without q")
        if q is not None:
            _check_half("q", q, k, k.dim())
            if q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
                raise RuntimeError("q and k must agree in tokens and head dim")
            if q_out is not None:
                _check_half("q_out", q_out, k, k.dim())
                if q_out.shape != q.shape:
                    raise RuntimeError("q_out must match q in shape")
        if rope is not None:
            _check("rope", rope, k, 2)
            if rope.dtype != torch.float32 or not rope.is_contiguous():
                raise RuntimeError("rope must be a contiguous fp32 table")
        p = _lib.AppendParams()
        p.k_stride[:], p.v_stride[:] = _token_strides(k), _token_strides(v)
        if q is not None:
            p.q_stride[:] = _token_strides(q)
            p.q_out_stride[:] = _token_strides(q_out if q_out is not None else torch.empty_like(q))
        p.k_cache_stride[:], p.v_cache_stride[:] = _page_strides(k_cache), _page_strides(v_cache)
        p.table_stride = block_table.stride(0) if B > 1 else block_table.shape[1]
        p.B, p.Hq, p.Hkv, p.D = B, q.shape[-2] if q is not None else 0, k.shape[-2], k.shape[-1]
        p.n, p.total = (k.shape[1], 0) if cu_q is None else (0, k.shape[0])
        if rope is not None:
            p.rot, p.rope_rows = min(rope.shape[1], _INT32_MAX), min(rope.shape[0], _INT32_MAX)
        p.interleaved = 1 if interleaved else 0
        p.page_size, p.n_pages, p.table_width = k_cache.shape[1], k_cache.shape[0], block_table.shape[1]
        p.dtype = _DTYPES[k.dtype]
        form = _keep(_append_forms, key, bytes(p)[_APPEND_POINTERS:])
    if q is not None and q_out is None:
        q_out = torch.empty_like(q)
    if k.numel() > 0:
        device = k.device
        status = _status_words.get(("cuda", device.index))
        block = _pack_append(
            k.data_ptr(), v.data_ptr(), 0 if q is None else q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            0 if q is None else q_out.data_ptr(), 0 if rope is None else rope.data_ptr(),
            (_status_word(device) if status is None else status).data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            0 if cu_q is None else cu_q.data_ptr()) + form
        if _current_device() == device.index:
            rc = _lib.lib.miniattn_paged_append(block, _current_raw_stream(device.index))
        else:
            with torch.cuda.device(device):
                rc = _lib.lib.miniattn_paged_append(block, _current_raw_stream(device.index))
        if rc != _lib.OK:
            _lib.check(rc, "miniattn_paged_append")
    return q_out


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    cu_q: Optional[torch.Tensor] = None,
    max_q: Optional[int] = None,
    window: Optional[int] = None,
    sinks: int = 0,
    shared_len: int = 0,
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
):
    """Causal attention of new tokens over the paged keys and values of their sequences, their own among them (conventions:
    module docstring): decode, drafts of a few tokens, chunked prefill, mixed batches.

    Query heads are a multiple of the cache's; KV head g serves query heads g*G..g*G+G-1.  A token sees the keys up to its own
    position; with ``window`` the last ``window`` of them and the first ``sinks`` tokens of its sequence.  Tokens that see none
    (padding) come out 0, their lse -inf.

    ``max_q``, with ``cu_q``: the most rows that one sequence has.  It picks the kernel and nothing else; without it the rows
    of ``q`` are taken for it.  ``shared_len``: the first ``shared_len`` tokens (whole pages) are the same for all sequences,
    the rows of the block table begin with the same pages.  Decode and drafts (up to 32 rows of a KV head: tokens of a sequence
    x query heads that share it) read them once for the whole batch where 100 MB would be read otherwise; other calls, and shorter
    prefixes, are read sequence by sequence.

    Returns ``out`` or ``(out, lse)``, lse fp32, the natural logarithm of the softmax denominators: (B, Hq, n), or (Hq, rows)
    with ``cu_q``.  A key that is NaN makes the rows that see it NaN, and no others.  A NaN or infinity among the *values* of a key
    that any row of a sequence sees may show in others of its rows, among those of a shared prefix in the rows of every
    sequence that holds some of its tokens.
    """
    if max_q is not None and type(max_q) is not int:
        max_q = _as_int("max_q", max_q)
    if window is not None and type(window) is not int:
        window = _as_int("window", window)
    if type(sinks) is not int:
        sinks = _as_int("sinks", sinks)
    if type(shared_len) is not int:
        shared_len = _as_int("shared_len", shared_len)
    if softmax_scale is not None and type(softmax_scale) is not float:
        softmax_scale = float(softmax_scale)
    try:
        key = (_form(q), _form(k_cache), _form(v_cache), _form(block_table), _form(seq_lens), _form(cu_q), _form(out), max_q,
               window, sinks, shared_len, softmax_scale)
        form = _attend_forms.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = form = None
    if form is None:
        _check_half("q", q, None, 4 if cu_q is None else 3)
        B = _check_paged(q, k_cache, v_cache, block_table, seq_lens, cu_q)
        Hq, Hkv = q.shape[-2], k_cache.shape[2]
        if Hkv == 0 or Hq % Hkv:
            raise RuntimeError(f"number of query heads ({Hq}) must be a multiple of KV heads ({Hkv})")
        if out is not None:
            _check_half("out", out, q, q.dim())
            if out.shape != q.shape:
                raise RuntimeError("out must match q in shape")
        p = _lib.CacheParams()
        # compared with null by the question for the scratch; what is launched gets its pointers below
        p.block_table, p.seq_lens, p.cu_q = block_table.data_ptr(), seq_lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr()
        p.q_stride[:] = _token_strides(q)
        p.o_stride[:] = _token_strides(out if out is not None else torch.empty_like(q))
        p.k_stride[:], p.v_stride[:] = _page_strides(k_cache), _page_strides(v_cache)
        p.table_stride = block_table.stride(0) if B > 1 else block_table.shape[1]
        p.B, p.Hq, p.Hkv, p.D = B, Hq, Hkv, q.shape[-1]
        if cu_q is None:
            p.Nq = q.shape[1]
            p.lse_stride[:] = (Hq * p.Nq, p.Nq)
        else:
            p.total_q = q.shape[0]
            p.Nq = min(_whole("max_q", max_q, 1), p.total_q) if max_q is not None else 0
            p.lse_stride[:] = (0, p.total_q)
        p.page_size, p.n_pages, p.table_width = k_cache.shape[1], k_cache.shape[0], block_table.shape[1]
        p.window = _whole("window", window, 1) if window is not None else 0
        p.sinks, p.shared_len = _whole("sinks", sinks, 0), _whole("shared_len", shared_len, 0)
        p.dtype = _DTYPES[q.dtype]
        p.softmax_scale = softmax_scale if softmax_scale is not None else 0.0
        need = _cache_scratch_bytes(p, q.device)
        lse_shape = (B, Hq, q.shape[1]) if cu_q is None else (Hq, q.shape[0])
        form = _keep(_attend_forms, key, (bytes(p)[_ATTEND_POINTERS:], need, lse_shape))
    rest, need, lse_shape = form
    if out is None:
        out = torch.empty_like(q)
    lse = torch.empty(lse_shape, dtype=torch.float32, device=q.device) if return_lse else None
    if q.numel() > 0:
        device = q.device
        status = _status_words.get(("cuda", device.index))
        _launch_cache(_pack_attend(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            (_status_word(device) if status is None else status).data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            0 if cu_q is None else cu_q.data_ptr()) + rest, need, device, shared_len > 0)
    return (out, lse) if return_lse else out
