"""Paged KV cache: pages of 16 to 128 positions handed to sequences through a page
table, held in bf16 or in E4M3 with one power-of-two scale per page and KV head.

``append`` rotates new query and key rows and stores keys and values;
``attention`` runs the causal attention of those rows over the cache, from one token
per sequence (decode) over a few (verification of drafted tokens) to whole prompts.
``PagedKvCache`` owns the pages and hands them out; ``batched.BatchedDecoder`` decodes
over one.  The reference keeps one dense slab per model instead
(``megakernels/llama.py:552-574``).

The functions take plain tensors:

* ``k_pages`` / ``v_pages``: ``[pages, kv_heads, page_size, head_dim]``, bf16 or
  ``float8_e4m3fn``, last dimension dense, the others at any pitch that is a multiple of
  16 bytes (a dense cache ``[batch, positions, kv_heads, head_dim]`` seen as pages works).
* ``k_scales`` / ``v_scales``: fp32 ``[pages, kv_heads]``, 8-bit caches only; a value is code times scale.
* ``page_table``: int32 ``[sequences, columns]``; a negative id means "no page".
* token rows ``[tokens, heads, head_dim]`` bf16, last dimension dense.  Sequence ``b`` owns rows
  ``cu_tokens[b] .. cu_tokens[b + 1] - 1``, or ``tokens / sequences`` rows each without ``cu_tokens``.

Nothing synchronises.  Page ids, positions and offsets live on the device and are checked there:
what lies outside its tensor is left out, and the next ``check_errors`` raises.
"""
from __future__ import annotations

import math

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


_error_words: dict = {}


def _error_word(device: torch.device) -> torch.Tensor:
    word = _error_words.get(device.index)
    if word is None:
        word = torch.zeros(1, dtype=torch.int32, device=device)
        _error_words[device.index] = word
    return word


def _cache_struct(k_pages, v_pages, k_scales, v_scales) -> _lib.MkPagedCache:
    dtype = k_pages.dtype
    if not k_pages.is_cuda or not v_pages.is_cuda:
        raise ValueError("k_pages and v_pages must be CUDA tensors")
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride() or v_pages.dtype != dtype:
        raise ValueError("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] tensors of one type, shape and layout")
    pages, heads, size, dim = k_pages.shape
    if dtype == torch.float8_e4m3fn:
        code = _lib.MK_CACHE_E4M3
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            if t is None or t.dtype != torch.float32 or t.shape != (pages, heads) or not t.is_contiguous() or t.device != k_pages.device:
                raise ValueError(f"{name} must be a contiguous fp32 [pages, kv_heads] tensor on the cache's device")
        scales = k_scales.data_ptr(), v_scales.data_ptr()
    elif dtype == torch.bfloat16:
        if k_scales is not None or v_scales is not None:
            raise ValueError("a bf16 cache has no scales")
        code, scales = _lib.MK_CACHE_BF16, (None, None)
    else:
        raise ValueError("the cache must be bf16 or float8_e4m3fn")
    page_stride, head_stride, slot_stride, last = k_pages.stride()
    if last != 1:
        raise ValueError("head_dim must be the dense dimension of the pages")
    # the pitch of a dimension of one element is never used; it only has to be a valid one
    if size == 1:
        slot_stride = dim
    if heads == 1:
        head_stride = size * slot_stride
    if pages == 1:
        page_stride = max(heads * head_stride, size * slot_stride)
    return _lib.MkPagedCache(k_pages.data_ptr(), v_pages.data_ptr(), *scales, page_stride, head_stride, slot_stride, code, pages, size, heads,
                             dim, 0)


def _int_vector(name, t, count, device):
    if t.dtype != torch.int32 or t.device != device or t.ndim != 1 or t.shape[0] != count or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of {count} elements on the cache's device")


def _batch_struct(page_table, where, name, cu_tokens, tokens, device) -> _lib.MkPagedBatch:
    if page_table.ndim != 2 or page_table.dtype != torch.int32 or page_table.device != device or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be an int32 [sequences, columns] tensor with dense rows on the cache's device")
    seqs, columns = page_table.shape
    _int_vector(name, where, seqs, device)
    if cu_tokens is not None:
        _int_vector("cu_tokens", cu_tokens, seqs + 1, device)
    elif seqs and tokens % seqs:
        raise ValueError(f"{tokens} rows do not divide over {seqs} sequences; give cu_tokens")
    return _lib.MkPagedBatch(page_table.data_ptr(), max(page_table.stride(0), columns) if seqs == 1 else page_table.stride(0), where.data_ptr(),
                             None if cu_tokens is None else cu_tokens.data_ptr(), _error_word(device).data_ptr(), seqs, tokens, columns, 0)


def _rows(name, t, heads, tokens, dim, device):
    if t.ndim != 3 or t.dtype != torch.bfloat16 or t.device != device or t.shape[2] != dim or t.stride(2) != 1 \
            or (heads is not None and t.shape[1] != heads) or (tokens is not None and t.shape[0] != tokens):
        raise ValueError(f"{name} must be a bf16 [{'tokens' if tokens is None else tokens}, "
                         f"{'heads' if heads is None else heads}, {dim}] tensor with dense rows on the cache's device")
    # a pitch that is never used (one token, one head) need not be a valid one
    return t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0


def _output(name, out, like, device):
    shape = tuple(like.shape)
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or out.device != device or tuple(out.shape) != shape or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bf16 tensor {list(shape)} on the cache's device")
    return out


class _on:
    """The device of a call as the current one (left alone where it is already)."""

    def __init__(self, device):
        self.device = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.device:
            torch.cuda.set_device(self.device)

    def __exit__(self, *exc):
        if self.before != self.device:
            torch.cuda.set_device(self.before)


def append(k, v, k_pages, v_pages, page_table, start, *, q=None, q_out=None, rope_cos=None, rope_sin=None, layout="interleaved",
           k_scales=None, v_scales=None, cu_tokens=None):
    """Store new key and value rows at positions ``start[b], start[b] + 1, ...`` of every sequence, keys (and
    queries) rotated on the way.  Returns the rotated ``q`` (``q_out`` if given), or None without ``q``.

    ``start``: int32 ``[sequences]``; a negative one marks an idle sequence, whose rows are neither stored nor
    rotated.  ``rope_cos`` / ``rope_sin``: fp32 ``[positions, rot]`` tables, ``rot`` a multiple of 16 up to
    ``head_dim`` (the rest of a head passes unchanged); ``layout`` "interleaved" pairs elements ``(2i, 2i + 1)``,
    "half" pairs ``(i, i + rot / 2)``.  Without tables nothing is rotated.

    8-bit pages: see the module's header and ``mk_paged_append`` for how a page's scale is chosen and grows.
    Sequences of one call must not share the pages they append to."""
    cache = _cache_struct(k_pages, v_pages, k_scales, v_scales)
    device, dim = k_pages.device, cache.head_dim
    tokens = k.shape[0]
    k_pitch, v_pitch = _rows("k", k, cache.num_kv_heads, None, dim, device), _rows("v", v, cache.num_kv_heads, tokens, dim, device)
    batch = _batch_struct(page_table, start, "start", cu_tokens, tokens, device)
    if layout not in ("interleaved", "half"):
        raise ValueError(f"layout must be 'interleaved' or 'half', got {layout!r}")
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos and rope_sin go together")
    cos = sin = None
    rot = positions = 0
    if rope_cos is not None:
        for name, t in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
            if t.ndim != 2 or t.dtype != torch.float32 or t.device != device or not t.is_contiguous() or t.shape != rope_cos.shape:
                raise ValueError(f"{name} must be a contiguous fp32 [positions, rot] tensor on the cache's device")
        positions, rot = rope_cos.shape
        cos, sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    q_pitch, q_ptr, out_ptr, heads = (0, 0), None, None, 0
    if q is not None:
        q_pitch, q_ptr, heads = _rows("q", q, None, tokens, dim, device), q.data_ptr(), q.shape[1]
        q_out = _output("q_out", q_out, q, device)
        out_ptr = q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    if tokens == 0:
        return q_out
    args = _lib.MkPagedAppend(q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, cos, sin, *q_pitch, *k_pitch, *v_pitch, heads, rot, positions,
                              1 if layout == "half" else 0)
    with _on(device):
        _lib.check(_lib.load().mk_paged_append(cache, batch, args, torch.cuda.current_stream(device).cuda_stream))
    return q_out


def attention(q, k_pages, v_pages, page_table, lengths, *, scale=None, k_scales=None, v_scales=None, cu_tokens=None, out=None,
              workspace=None):
    """Causal attention of the newest rows of every sequence over its cache, which already holds their keys and
    values: row ``i`` of sequence ``b``'s ``n`` rows sees positions ``0 .. lengths[b] - n + i``.  ``q`` is
    ``[tokens, heads, head_dim]`` with heads a multiple of the cache's; returns ``out`` of the same shape, bf16.

    ``lengths``: int32 ``[sequences]``, the new rows included.  A row that sees no position (an idle sequence of
    length 0) becomes zero; rows outside every sequence stay as they were in ``out``.  ``scale`` defaults to
    ``1 / sqrt(head_dim)``.  ``workspace``: a uint8 tensor of ``attention_workspace`` bytes for callers that
    allocate once; calls that may overlap in time need their own."""
    cache = _cache_struct(k_pages, v_pages, k_scales, v_scales)
    device = k_pages.device
    q_pitch = _rows("q", q, None, None, cache.head_dim, device)
    tokens, heads = q.shape[0], q.shape[1]
    batch = _batch_struct(page_table, lengths, "lengths", cu_tokens, tokens, device)
    out = _output("out", out, q, device)
    if tokens == 0:
        return out
    lib = _lib.load()
    with _on(device):
        if workspace is None:
            need = _workspace_bytes(cache, batch, heads)
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
        elif workspace.device != device or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous tensor on the cache's device")
        args = _lib.MkPagedAttention(q.data_ptr(), out.data_ptr(), None if workspace is None else workspace.data_ptr(),
                                     0 if workspace is None else workspace.numel() * workspace.element_size(), *q_pitch, heads,
                                     1 / math.sqrt(cache.head_dim) if scale is None else scale)
        _lib.check(lib.mk_paged_attention(cache, batch, args, torch.cuda.current_stream(device).cuda_stream))
    return out


def attention_workspace(q, k_pages, v_pages, page_table, lengths, *, k_scales=None, v_scales=None, cu_tokens=None) -> int:
    """Bytes of workspace that ``attention`` needs for these sizes (the tensors' contents do not matter)."""
    cache = _cache_struct(k_pages, v_pages, k_scales, v_scales)
    batch = _batch_struct(page_table, lengths, "lengths", cu_tokens, q.shape[0], k_pages.device)
    with _on(k_pages.device):
        return _workspace_bytes(cache, batch, q.shape[1])


def _workspace_bytes(cache, batch, heads) -> int:
    lib = _lib.load()
    need = lib.mk_paged_attention_workspace(cache, batch, heads)
    if need < 0:
        raise _lib.MegakernelError(_lib.MK_ERR_UNSUPPORTED, lib.mk_last_error().decode())
    return need


def check_errors(device=None) -> None:
    """Synchronises and raises if a paged call met a page id, position, length or row offset outside its tensor,
    or if a bounded wait inside a kernel ran out."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    torch.cuda.synchronize(device)
    word = _error_word(device)
    value = int(word.item())
    if value:
        word.zero_()
        if value & 1:
            raise _lib.MegakernelError(_lib.MK_ERR_DEVICE_WAIT, "a bounded wait inside a kernel ran out")
        raise _lib.MegakernelError(_lib.MK_ERR_BAD_ARGUMENT, "a page id, position, length or row offset given to a paged call was outside its tensor; it was left out")
