"""Attention of new tokens over a paged cache of keys and values, and the cache itself.

``csr_attention_forward`` computes all rows of an attention pattern at once.  A model that answers token by
token has one new query a sequence and keeps the keys and values of the tokens before it; here they lie in
pages of a fixed number of tokens, and the page table is a CSR pattern of its own: row = sequence, column =
page id, in the order of the tokens.

    paged_cache_write     keys and values of new tokens into their slots, quantised on the way if the pages are 8-bit
    paged_cache_read      tokens out of their slots again
    csr_paged_attention   one new token of every sequence attends to the tokens of its pages

Pages are ``[n_pages, page_size, n_kv_heads, head_dim]`` tensors, one for keys and one for values, in float32,
bfloat16, float16, ``float8_e4m3fn`` or int8, with any strides whose features are contiguous.  The two 8-bit types
go with float32 scales ``[n_pages, n_kv_heads, page_size]``, one for each row of ``head_dim`` features: value =
code * scale.  A slot is ``page * page_size + place in the page``.

These are operators of inference: they have no backward and no forward-mode derivative, and a call that would need one is
refused.  The reference has no counterpart (its attention, ``autosage/_auto.py:762-780``, is the whole-pattern form).
"""
from __future__ import annotations

import os
from typing import Optional

import torch
from torch._subclasses.fake_tensor import FakeTensor
from torch.autograd import forward_ad

from . import _native, ops

_WIDE = (torch.float32, torch.bfloat16, torch.float16)
_CODED = (torch.float8_e4m3fn, torch.int8)
MAX_HEAD_DIM = 256


def _index(name: str, tensor: torch.Tensor, device: torch.device) -> torch.Tensor:
    dtype = tensor.dtype
    if dtype is not torch.int64 and dtype is not torch.int32:
        raise TypeError(f"{name} must use integer indices")
    if tensor.dim() != 1:
        raise ValueError(f"{name} must be one-dimensional")
    if tensor.device != device:
        raise ValueError(f"{name} must be on the device of the pages")
    if dtype is not torch.int64:
        tensor = tensor.to(torch.int64)
    return tensor if tensor.is_contiguous() else tensor.contiguous()


def _refuse_pages(key_pages, value_pages, key_scales, value_scales) -> None:
    """Says what is wrong with the pages."""
    if key_pages.ndim != 4 or key_pages.shape != value_pages.shape:
        raise ValueError("key_pages and value_pages must have the same [n_pages, page_size, n_kv_heads, head_dim] shape")
    n_pages, page_size, heads, dim = key_pages.shape
    if min(page_size, heads, dim) < 1:
        raise ValueError("page_size, n_kv_heads and head_dim must be positive")
    if dim > MAX_HEAD_DIM:
        raise ValueError(f"head_dim is at most {MAX_HEAD_DIM}")
    dtype, device = key_pages.dtype, key_pages.device
    if dtype != value_pages.dtype or dtype not in _native.TYPES:
        raise TypeError("the pages must both be float32, bfloat16, float16, float8_e4m3fn or int8")
    if dim > 1 and (key_pages.stride(3) != 1 or value_pages.stride(3) != 1):
        raise ValueError("the features of a page row must be contiguous")
    if value_pages.device != device:
        raise ValueError("key_pages and value_pages must be on the same device")
    if dtype not in _CODED:
        raise ValueError("scales go with 8-bit pages only")
    for name, scales in (("key_scales", key_scales), ("value_scales", value_scales)):
        if scales is None:
            raise ValueError(f"8-bit pages need {name}")
        if scales.dtype != torch.float32:
            raise TypeError(f"{name} must be float32")
        if scales.shape != (n_pages, heads, page_size):
            raise ValueError(f"{name} must have shape [n_pages, n_kv_heads, page_size]")
        if scales.device != device:
            raise ValueError(f"{name} must be on the device of the pages")
    raise AssertionError("pages refused for no reason")


def _check_pages(key_pages, value_pages, key_scales, value_scales) -> torch.Size:
    """Checks the pages and returns their shape (n_pages, page_size, heads, dim)."""
    shape, dtype, device = key_pages.shape, key_pages.dtype, key_pages.device
    fine = (len(shape) == 4 and shape == value_pages.shape and shape[1] > 0 and shape[2] > 0 and 0 < shape[3] <= MAX_HEAD_DIM
            and value_pages.dtype is dtype and value_pages.device == device
            and ((key_pages.stride()[3] == 1 and value_pages.stride()[3] == 1) or shape[3] == 1))
    if fine and _native.TYPES.get(dtype, 9) <= 2:
        fine = key_scales is None and value_scales is None
    elif fine:
        wanted = (shape[0], shape[2], shape[1])
        fine = (dtype in _CODED and key_scales is not None and value_scales is not None
                and key_scales.dtype is torch.float32 and value_scales.dtype is torch.float32
                and key_scales.shape == wanted and value_scales.shape == wanted
                and key_scales.device == device and value_scales.device == device)
    if not fine:
        _refuse_pages(key_pages, value_pages, key_scales, value_scales)
    return shape


def _require_native(device: torch.device, *tensors: Optional[torch.Tensor]) -> None:
    grad = torch.is_grad_enabled()
    for tensor in tensors:
        if tensor is None:
            continue
        if grad and tensor.requires_grad:
            raise RuntimeError("the paged cache has no backward; call it under torch.no_grad() or detach its inputs")
        if type(tensor) is FakeTensor:   # its address is 0, and a workspace made beside it would be one too
            raise RuntimeError("the paged cache needs tensors with memory, not fake ones")
    if forward_ad._current_level >= 0:   # (no_grad() does not end forward mode)
        for tensor in tensors:
            if tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None:
                raise RuntimeError("the paged cache has no forward-mode derivative; call it with the primal parts of its inputs")
    if device.type != "cuda":
        raise RuntimeError("the paged cache needs CUDA tensors")
    if _native._LIB is None and not ops.load_native():
        detail = f": {ops.native_load_error()}" if ops.native_load_error() else ""
        raise RuntimeError(f"AutoSAGE CUDA extension is unavailable{detail}")


def _contiguous_features(rows: torch.Tensor) -> torch.Tensor:
    return rows if rows.stride(2) == 1 or rows.size(2) <= 1 else rows.contiguous()


def _checking() -> bool:
    return os.environ.get("AUTOSAGE_CHECK_INDICES") == "1"


def _check_writable(*tensors: Optional[torch.Tensor]) -> None:
    for i, tensor in enumerate(tensors):
        if tensor is not None and 0 in tensor.stride() and any(
                step == 0 and size > 1 for step, size in zip(tensor.stride(), tensor.shape)):
            name = ("key_pages", "value_pages", "key_scales", "value_scales")[i]
            raise ValueError(f"{name} is written and must not repeat memory (it has a stride of 0)")


def paged_cache_write(slots: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
                      value_pages: torch.Tensor, *, key_scales: Optional[torch.Tensor] = None,
                      value_scales: Optional[torch.Tensor] = None) -> None:
    """Writes token t of ``key`` and ``value`` (``[T, n_kv_heads, head_dim]``) to slot ``slots[t]`` of the pages, in place.

    Pages have the type of the tokens, or an 8-bit type: then ``scale = max|x| / 448`` (e4m3) or ``/ 127`` (int8) over
    the features of a row, and each code is the nearest to ``x / scale``, ties to even.  A row with an infinity or a
    NaN reads back as NaN.

    A slot outside the pages (-1, say) is skipped: padding.  The others must differ from one another: of two tokens
    with the same slot, what is kept is a mixture (``AUTOSAGE_CHECK_INDICES=1`` refuses such a call).  Neither ``key`` and
    ``value`` nor other pages or scales of the call share memory with the slots that are written."""
    n_pages, page_size, heads, dim = _check_pages(key_pages, value_pages, key_scales, value_scales)
    shape = key.shape
    if len(shape) != 3 or shape != value.shape or shape[1] != heads or shape[2] != dim:
        raise ValueError("key and value must have the same [tokens, n_kv_heads, head_dim] shape, as wide as the pages")
    if key.dtype != value.dtype or key.dtype not in _WIDE:
        raise TypeError("key and value must both be float32, bfloat16 or float16")
    if key_pages.dtype not in _CODED and key_pages.dtype != key.dtype:
        raise TypeError("the pages must have the type of key and value, or an 8-bit type")
    device = key_pages.device
    if key.device != device or value.device != device:
        raise ValueError("key and value must be on the device of the pages")
    slots = _index("slots", slots, device)
    if slots.numel() != shape[0]:
        raise ValueError("slots must contain one slot per token")
    _check_writable(key_pages, value_pages, key_scales, value_scales)
    _require_native(device, key, value, key_pages, value_pages, key_scales, value_scales)
    if slots.numel() == 0 or n_pages == 0:
        return
    if _checking():
        kept = slots[(slots >= 0) & (slots < n_pages * page_size)]
        if kept.unique().numel() != kept.numel():
            raise RuntimeError("two tokens have the same slot")
    _native.paged_cache_write(slots, _contiguous_features(key), _contiguous_features(value), key_pages, value_pages,
                              key_scales, value_scales)
    # as after any operation in place; tensors made in inference mode keep no count
    written = (key_pages, value_pages) if key_scales is None else (key_pages, value_pages, key_scales, value_scales)
    for tensor in written:
        if tensor.is_inference():
            written = [tensor for tensor in written if not tensor.is_inference()]
            break
    torch.autograd.graph.increment_version(written)


def paged_cache_read(slots: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, *,
                     key_scales: Optional[torch.Tensor] = None, value_scales: Optional[torch.Tensor] = None,
                     dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values in the slots ``slots``, as two ``[T, n_kv_heads, head_dim]`` tensors of type ``dtype`` (that
    of the pages, or float32 for 8-bit pages).  Slots may repeat; one outside the pages reads as zeros."""
    _, _, heads, dim = _check_pages(key_pages, value_pages, key_scales, value_scales)
    if dtype is None:
        dtype = torch.float32 if key_pages.dtype in _CODED else key_pages.dtype
    if dtype not in _WIDE:
        raise TypeError("dtype must be float32, bfloat16 or float16")
    device = key_pages.device
    slots = _index("slots", slots, device)
    _require_native(device, key_pages, value_pages, key_scales, value_scales)
    tokens = slots.numel()
    key = slots.new_empty((tokens, heads, dim), dtype=dtype)
    value = torch.empty_like(key)
    if tokens:
        _native.paged_cache_read(slots, key, value, key_pages, value_pages, key_scales, value_scales)
    return key, value


def _debug_check_table(crow, col, lengths, n_pages: int, page_size: int) -> None:
    """AUTOSAGE_CHECK_INDICES=1: verify the page table before the launch (synchronises)."""
    if int(crow[0].item()) != 0 or int(crow[-1].item()) != col.numel():
        raise RuntimeError("crow must run from 0 to the number of columns")
    pages = crow[1:] - crow[:-1]
    if bool((pages < 0).any().item()):
        raise RuntimeError("crow must be non-decreasing")
    if bool(((lengths < 0) | (lengths > pages * page_size)).any().item()):
        raise RuntimeError("lengths must lie between 0 and what the pages of the row hold")
    if col.numel() and int(col.max().item()) >= n_pages:
        raise RuntimeError(f"page ids must lie below {n_pages}")


def csr_paged_attention(crow: torch.Tensor, col: torch.Tensor, lengths: torch.Tensor, query: torch.Tensor,
                        key_pages: torch.Tensor, value_pages: torch.Tensor, *,
                        key_scales: Optional[torch.Tensor] = None, value_scales: Optional[torch.Tensor] = None,
                        scale: Optional[float] = None, window: Optional[int] = None, return_lse: bool = False):
    """``softmax_t(scale * <query, k_t>) v_t`` for one new token of every sequence.

    ``crow`` ``[B + 1]`` and ``col`` are the page table in CSR form (row r owns the pages ``col[crow[r]:crow[r + 1]]``, in
    the order of its tokens) and ``lengths`` ``[B]`` the number of tokens of each row, at most what its pages hold.  ``query``
    is ``[B, n_heads, head_dim]`` with ``n_heads`` a multiple of the pages' ``n_kv_heads``: neighbouring query heads
    share a key head.  Pages have the type of the query, or an 8-bit type.  ``scale=None`` leaves the scores unscaled, as in
    ``csr_attention_forward``; ``window=w`` lets a token see the last w tokens of its row only.

    Returns ``[B, n_heads, head_dim]`` in the type of the query and, with ``return_lse=True``, the natural
    logarithm of each softmax's denominator as float32 ``[B, n_heads]`` (parts computed over different pages can be
    joined with it).  A row that sees nothing gives 0 and ``-inf``.  A page id outside the pages is a hole whose
    tokens are not seen (``AUTOSAGE_CHECK_INDICES=1`` takes only negative ids for one); whatever lies behind a row's length
    in its last pages is not read.  An infinity among the values that are seen makes its feature infinite, unless its weight is
    one that float32 calls 0: then NaN, as 0 times infinity."""
    n_pages, page_size, kv_heads, dim = _check_pages(key_pages, value_pages, key_scales, value_scales)
    device = key_pages.device
    shape = query.shape
    if len(shape) != 3 or shape[2] != dim:
        raise ValueError("query must have shape [rows, n_heads, head_dim] with the pages' head_dim")
    rows, heads, _ = shape
    if heads < 1 or heads % kv_heads != 0:
        raise ValueError("n_heads must be a positive multiple of n_kv_heads")
    if query.dtype not in _WIDE:
        raise TypeError("query must be float32, bfloat16 or float16")
    if key_pages.dtype not in _CODED and key_pages.dtype != query.dtype:
        raise TypeError("the pages must have the type of the query, or an 8-bit type")
    if query.device != device:
        raise ValueError("query must be on the device of the pages")
    crow, col, lengths = _index("crow", crow, device), _index("col", col, device), _index("lengths", lengths, device)
    if crow.numel() != rows + 1:
        raise ValueError("crow must contain one entry per row and one more")
    if lengths.numel() != rows:
        raise ValueError("lengths must contain one entry per row")
    if window is not None:
        if not isinstance(window, int):
            raise TypeError("window must be a whole number of tokens")
        if window < 1:
            raise ValueError("window must be positive")
    _require_native(device, query, key_pages, value_pages, key_scales, value_scales)
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    lse = query.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    if rows:
        if _checking():
            _debug_check_table(crow, col, lengths, n_pages, page_size)
        _native.paged_attention(crow, col, lengths, _contiguous_features(query), out, lse, key_pages, value_pages, key_scales,
                                value_scales, 1.0 if scale is None else float(scale), 0 if window is None else min(window, 1 << 62))
    return (out, lse) if return_lse else out


__all__ = ["csr_paged_attention", "paged_cache_read", "paged_cache_write"]
