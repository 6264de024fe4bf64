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

import ctypes as C
import struct
from functools import lru_cache

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


_error_words: dict = {}


def _error_word(device: int) -> torch.Tensor:
    word = _error_words.get(device)
    if word is None:
        word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", device))
        _error_words[device] = word
    return word


# The structs of include/b200_megakernel.h as bytes: packing them costs a fraction of filling ctypes fields, and a
# decode step makes these calls for every layer.
_CACHE = struct.Struct("=4Q3q6i")       # MkPagedCache
_BATCH = struct.Struct("=QqQQQ4i")      # MkPagedBatch
_APPEND = struct.Struct("=6Q6q4i")      # MkPagedAppend
_ATTENTION = struct.Struct("=3Qq2qif")  # MkPagedAttention


@lru_cache(maxsize=1)
def _entry_points():
    lib = _lib.load()
    assert (_CACHE.size, _BATCH.size, _APPEND.size, _ATTENTION.size) == tuple(lib.mk_abi_sizeof(i) for i in range(4, 8))
    call = C.CFUNCTYPE(C.c_int, C.c_char_p, C.c_char_p, C.c_char_p, C.c_void_p)
    size = C.CFUNCTYPE(C.c_int64, C.c_char_p, C.c_char_p, C.c_int32)
    return (call(("mk_paged_append", lib)), call(("mk_paged_attention", lib)), size(("mk_paged_attention_workspace", lib)))


def _cache_bytes(k_pages, v_pages, k_scales, v_scales):
    """(packed MkPagedCache, device index, KV heads, head_dim)"""
    if not k_pages.is_cuda or not v_pages.is_cuda:
        raise ValueError("k_pages and v_pages must be CUDA tensors")
    device, dtype, shape, strides = k_pages.get_device(), k_pages.dtype, k_pages.shape, k_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.stride() != strides or v_pages.dtype is not dtype or v_pages.get_device() != device:
        raise ValueError("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] tensors of one type, shape and layout on one device")
    pages, heads, size, dim = shape
    page_stride, head_stride, slot_stride, last = strides
    if dtype is torch.float8_e4m3fn:
        code = _lib.MK_CACHE_E4M3
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            if t is None or t.dtype is not torch.float32 or t.shape != (pages, heads) or not t.is_contiguous() or t.get_device() != device:
                raise ValueError(f"{name} must be a contiguous fp32 [pages, kv_heads] tensor on the cache's device")
        ks, vs = k_scales.data_ptr(), v_scales.data_ptr()
    elif dtype is torch.bfloat16:
        if k_scales is not None or v_scales is not None:
            raise ValueError("a bf16 cache has no scales")
        code, ks, vs = _lib.MK_CACHE_BF16, 0, 0
    else:
        raise ValueError("the cache must be bf16 or float8_e4m3fn")
    if last != 1:
        raise ValueError("head_dim must be the dense dimension of the pages")
    # the pitch of a dimension of one element is never used; it only has to be a valid one
    if heads == 1:
        head_stride = size * slot_stride
    if pages == 1:
        page_stride = max(heads * head_stride, size * slot_stride)
    return _CACHE.pack(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, page_stride, head_stride, slot_stride, code, pages, size, heads, dim,
                       0), device, heads, dim


def _batch_bytes(page_table, where, name, cu_tokens, tokens, device):
    shape = page_table.shape
    if len(shape) != 2 or page_table.dtype is not torch.int32 or page_table.get_device() != device:
        raise ValueError("page_table must be an int32 [sequences, columns] tensor on the cache's device")
    seqs, columns = shape
    row, last = page_table.stride()
    if columns > 1 and last != 1:
        raise ValueError("page_table must have dense rows")
    if where.dtype is not torch.int32 or where.get_device() != device or where.shape != (seqs,) or not where.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of {seqs} elements on the cache's device")
    cu = 0
    if cu_tokens is not None:
        if cu_tokens.dtype is not torch.int32 or cu_tokens.get_device() != device or cu_tokens.shape != (seqs + 1,) or not cu_tokens.is_contiguous():
            raise ValueError(f"cu_tokens must be a contiguous int32 vector of {seqs + 1} elements on the cache's device")
        cu = cu_tokens.data_ptr()
    elif seqs and tokens % seqs:
        raise ValueError(f"{tokens} rows do not divide over {seqs} sequences; give cu_tokens")
    word = _error_words.get(device)
    if word is None:
        word = _error_word(device)
    return _BATCH.pack(page_table.data_ptr(), columns if seqs == 1 else row, where.data_ptr(), cu, word.data_ptr(), seqs, tokens, columns, 0)


def _rows(name, t, heads, tokens, dim, device):
    """(token pitch, head pitch) of bf16 rows; a pitch that is never used (one token, one head) need not be a valid one."""
    shape = t.shape
    if len(shape) != 3 or t.dtype is not torch.bfloat16 or t.get_device() != device or shape[2] != dim \
            or (heads is not None and shape[1] != heads) or (tokens is not None and shape[0] != tokens):
        raise ValueError(f"{name} must be a bf16 [{'tokens' if tokens is None else tokens}, "
                         f"{'heads' if heads is None else heads}, {dim}] tensor on the cache's device")
    token, head, last = t.stride()
    if last != 1:
        raise ValueError(f"{name} must have dense rows")
    return token if shape[0] > 1 else 0, head if shape[1] > 1 else 0


def _output(name, out, like, device):
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if out.dtype is not torch.bfloat16 or out.get_device() != device or out.shape != like.shape or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bf16 tensor {list(like.shape)} on the cache's device")
    return out


def _call(entry, device, *structs):
    """``entry`` on the device's current stream, with the device as the current one."""
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch._C._cuda_getDevice() == device:
        code = entry(*structs, stream)
    else:
        with torch.cuda.device(device):
            code = entry(*structs, stream)
    if code:
        _lib.check(code)


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
    cache, device, kv_heads, dim = _cache_bytes(k_pages, v_pages, k_scales, v_scales)
    tokens = k.shape[0]
    k_pitch, v_pitch = _rows("k", k, kv_heads, None, dim, device), _rows("v", v, kv_heads, tokens, dim, device)
    batch = _batch_bytes(page_table, start, "start", cu_tokens, tokens, device)
    if layout != "interleaved" and layout != "half":
        raise ValueError(f"layout must be 'interleaved' or 'half', got {layout!r}")
    cos = sin = rot = positions = 0
    if rope_cos is not None and rope_sin is not None:
        shape = rope_cos.shape
        for name, t in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
            if len(shape) != 2 or t.dtype is not torch.float32 or t.get_device() != device or not t.is_contiguous() or t.shape != shape:
                raise ValueError(f"{name} must be a contiguous fp32 [positions, rot] tensor on the cache's device")
        positions, rot = shape
        cos, sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    elif rope_cos is not None or rope_sin is not None:
        raise ValueError("rope_cos and rope_sin go together")
    q_pitch, q_ptr, out_ptr, heads = (0, 0), 0, 0, 0
    if q is not None:
        q_pitch, q_ptr, heads = _rows("q", q, None, tokens, dim, device), q.data_ptr(), q.shape[1]
        q_out = _output("q_out", q_out, q, device)
        out_ptr = q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    if tokens:
        args = _APPEND.pack(q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, cos, sin, *q_pitch, *k_pitch, *v_pitch, heads, rot, positions,
                            layout == "half")
        _call(_entry_points()[0], device, cache, batch, args)
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
    cache, device, _, dim = _cache_bytes(k_pages, v_pages, k_scales, v_scales)
    pitch = _rows("q", q, None, None, dim, device)
    tokens, heads = q.shape[0], q.shape[1]
    batch = _batch_bytes(page_table, lengths, "lengths", cu_tokens, tokens, device)
    out = _output("out", out, q, device)
    if tokens == 0:
        return out
    ws = ws_bytes = 0
    if workspace is None:
        ws_bytes = _workspace_bytes(cache, batch, heads, device)
        if ws_bytes:
            workspace = page_table.new_empty(ws_bytes >> 2)   # int32, on the same device
            ws = workspace.data_ptr()
    elif workspace.get_device() != device or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on the cache's device")
    else:
        ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), ws, ws_bytes, *pitch, heads, dim ** -0.5 if scale is None else scale)
    _call(_entry_points()[1], device, cache, batch, args)
    return out


def attention_workspace(q, k_pages, v_pages, page_table, lengths, *, k_scales=None, v_scales=None, cu_tokens=None) -> int:
    """Bytes of workspace that ``attention`` needs for these sizes (the tensors' contents do not matter)."""
    cache, device, _, _ = _cache_bytes(k_pages, v_pages, k_scales, v_scales)
    return _workspace_bytes(cache, _batch_bytes(page_table, lengths, "lengths", cu_tokens, q.shape[0], device), q.shape[1], device)


def _workspace_bytes(cache, batch, heads, device) -> int:
    if torch._C._cuda_getDevice() == device:
        need = _entry_points()[2](cache, batch, heads)
    else:
        with torch.cuda.device(device):
            need = _entry_points()[2](cache, batch, heads)
    if need < 0:
        raise _lib.MegakernelError(_lib.MK_ERR_UNSUPPORTED, _lib.load().mk_last_error().decode())
    return need


def check_errors(device=None) -> None:
    """Synchronises and raises if a paged call met a page id, position, length or row offset outside its tensor,
    or if a bounded wait inside a kernel ran out."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    torch.cuda.synchronize(index)
    word = _error_word(index)
    value = int(word.item())
    if value:
        word.zero_()
        if value & 1:
            raise _lib.MegakernelError(_lib.MK_ERR_DEVICE_WAIT, "a bounded wait inside a kernel ran out")
        raise _lib.MegakernelError(_lib.MK_ERR_BAD_ARGUMENT, "a page id, position, length or row offset given to a paged call was outside its tensor; it was left out")
