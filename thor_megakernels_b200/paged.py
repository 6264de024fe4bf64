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
  Finite and not negative; value scales that one row sees within a factor of 2^100 of one another.
* ``page_table``: int32 ``[sequences, columns]``; a negative id means "no page".
* token rows ``[tokens, heads, head_dim]`` bf16, last dimension dense.  Sequence ``b`` owns rows
  ``cu_tokens[b] .. cu_tokens[b + 1] - 1``, or ``tokens / sequences`` rows each without ``cu_tokens``.

For inference: results carry no gradient.  Nothing synchronises.  Page ids, positions and offsets live on the device and are checked there:
what lies outside its tensor is left out, and the next ``check_errors`` raises.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache

import torch

from . import _lib
from . import build as _build

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


_error_words: dict = {}


@lru_cache(maxsize=1)
def _binding():
    """The module of ``csrc/paged_binding.cpp``, bound to the library; there is no other path."""
    lib = _lib.load()
    try:
        _build.build_binding()
    except Exception as exc:  # one built from other sources, or for another torch or Python, is not used
        raise RuntimeError(f"_paged_binding.so is missing or of another build and could not be built ({exc}); "
                           "run `python -m thor_megakernels_b200.build`") from exc
    from . import _paged_binding

    _paged_binding.init(*(C.cast(getattr(lib, name), C.c_void_p).value
                          for name in ("mk_paged_append", "mk_paged_attention", "mk_paged_attention_workspace")),
                        *(lib.mk_abi_sizeof(which) for which in (4, 5, 6, 7)))
    return _paged_binding


def _error_word(device: int) -> torch.Tensor:
    word = _error_words.get(device)
    if word is None:
        # it outlives every graph, so it must not come from a graph's memory
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first paged call on a device cannot be captured in a CUDA graph: make one before (check_errors will do)")
        word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", device))
        torch.cuda.current_stream(device).synchronize()
        _binding().set_error_word(device, word.data_ptr())
        _error_words[device] = word
    return word


def _result(value, call, pages, args):
    """``value`` unless it is an int: the first call on a device is made again, anything else is the library's refusal."""
    if type(value) is int and value == -1:
        _error_word(pages.get_device())
        value = call(*args)
    if type(value) is int:
        _lib.check(value)
    return value


def append(k, v, k_pages, v_pages, page_table, start, *, q=None, q_out=None, rope_cos=None, rope_sin=None, layout="interleaved",
           k_scales=None, v_scales=None, cu_tokens=None):
    """Store new key and value rows at positions ``start[b], start[b] + 1, ...`` of every sequence, keys (and
    queries) rotated on the way.  Returns the rotated ``q`` (``q_out`` if given; it may be ``q`` itself), or None
    without ``q``.

    ``start``: int32 ``[sequences]``; a negative one marks an idle sequence, whose rows are neither stored nor
    rotated.  ``rope_cos`` / ``rope_sin``: fp32 ``[positions, rot]`` tables, ``rot`` a multiple of 16 up to
    ``head_dim`` (the rest of a head passes unchanged); ``layout`` "interleaved" pairs elements ``(2i, 2i + 1)``,
    "half" pairs ``(i, i + rot / 2)``.  Rows at positions beyond the tables are left out and reported.  Without
    tables nothing is rotated.

    8-bit pages: see the module's header and ``mk_paged_append`` for how a page's scale is chosen and grows.
    A page that a call appends to must stand in one place of the sequences' tables only."""
    if layout != "interleaved" and layout != "half":
        raise ValueError(f"layout must be 'interleaved' or 'half', got {layout!r}")
    call = _binding().append
    args = (k, v, k_pages, v_pages, page_table, start, q, q_out, rope_cos, rope_sin, layout == "half", k_scales, v_scales, cu_tokens)
    value = call(*args)
    return _result(value, call, k_pages, args) if type(value) is int else value


def attention(q, k_pages, v_pages, page_table, lengths, *, scale=None, k_scales=None, v_scales=None, cu_tokens=None, out=None,
              workspace=None):
    """Causal attention of the newest rows of every sequence over its cache, which already holds their keys and
    values: row ``i`` of sequence ``b``'s ``n`` rows sees positions ``0 .. lengths[b] - n + i``.  ``q`` is
    ``[tokens, heads, head_dim]`` with heads a multiple of the cache's; returns ``out`` of the same shape, bf16.

    ``lengths``: int32 ``[sequences]``, the new rows included.  A row that sees no position (an idle sequence of
    length 0) becomes zero; rows outside every sequence stay as they were in ``out``, which must not overlap ``q``.
    Scores, statistics and sums are fp32; how the softmax weights are rounded stands at ``mk_paged_attention``.
    ``scale`` defaults to ``1 / sqrt(head_dim)``.  ``workspace``: a uint8 tensor of ``attention_workspace`` bytes for
    callers that allocate once; calls that may overlap in time need their own."""
    call = _binding().attention
    args = (q, k_pages, v_pages, page_table, lengths, scale, k_scales, v_scales, cu_tokens, out, workspace)
    value = call(*args)
    return _result(value, call, k_pages, args) if type(value) is int else value


def attention_workspace(q, k_pages, v_pages, page_table, lengths, *, k_scales=None, v_scales=None, cu_tokens=None) -> int:
    """Bytes of workspace that ``attention`` needs for these sizes (the tensors' contents do not matter)."""
    call = _binding().attention_workspace
    args = (q, k_pages, v_pages, page_table, lengths, k_scales, v_scales, cu_tokens)
    return int(_result(call(*args), call, k_pages, args))


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
        torch.cuda.synchronize(index)   # or it could wipe out what a later call on another stream reports
        if value & 1:
            raise _lib.MegakernelError(_lib.MK_ERR_DEVICE_WAIT, "a bounded wait inside a kernel ran out")
        raise _lib.MegakernelError(_lib.MK_ERR_BAD_ARGUMENT, "a page id, position, length or row offset given to a paged call was outside its tensor; it was left out")


class PagedKvCache:
    """The pages of a model and who has them.

    ``k`` / ``v`` ``[layers, pages, kv_heads, page_size, head_dim]``, ``k_scales`` / ``v_scales`` ``[layers, pages, kv_heads]``
    (8-bit only), ``page_table`` int32 ``[max_seqs, max_pages]`` on the device, -1 where a sequence has no page.  A page id stands
    for the same place in every layer.  ``reserve`` before a call that reaches new positions, ``release`` when a sequence is done;
    both change the table in stream order (the current stream of the device), so a step that is queued already keeps its pages'
    ids, and a captured step sees the table as it is when it is replayed.  Neither can be captured itself."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, *, page_size: int = 64, max_seqs: int = 128,
                 max_positions: int | None = None, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}")
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError("the cache must be bf16 or float8_e4m3fn")
        if min(num_layers, num_pages, num_kv_heads, max_seqs, 1 if max_positions is None else max_positions) < 1:
            raise ValueError("layers, pages, heads, sequences and positions must be positive")
        self.page_size, self.num_pages = page_size, num_pages
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        # what a page holds before its first row is never read
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scales = self.v_scales = None
        if dtype == torch.float8_e4m3fn:
            self.k_scales, self.v_scales = (torch.ones(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
        columns = num_pages if max_positions is None else -(-max_positions // page_size)
        self.page_table = torch.full((max_seqs, columns), -1, dtype=torch.int32, device=device)
        if self.k.is_cuda:
            _error_word(self.k.get_device())   # so that the first call may be a captured one
        self._free = list(range(num_pages - 1, -1, -1))
        self._owned: list[list[int]] = [[] for _ in range(max_seqs)]

    @classmethod
    def for_model(cls, model, num_pages: int, **kwargs) -> "PagedKvCache":
        """A cache with the layers and heads of a model container."""
        cfg = model.config
        return cls(cfg.num_hidden_layers, num_pages, cfg.num_key_value_heads, cfg.head_dim, device=kwargs.pop("device", model.device), **kwargs)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _check(self, seq: int) -> None:
        if not 0 <= seq < len(self._owned):   # a negative index would be another sequence's
            raise IndexError(f"the cache has sequences 0 .. {len(self._owned) - 1}, got {seq}")
        if self.page_table.is_cuda:
            with torch.cuda.device(self.page_table.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("pages are handed out and taken back by the host: not inside a CUDA graph's capture")

    def reserve(self, seq: int, positions: int) -> None:
        """Give sequence ``seq`` pages for positions ``0 .. positions - 1`` (those it has stay its own)."""
        self._check(seq)
        owned = self._owned[seq]
        need = -(-positions // self.page_size)
        if need > self.page_table.shape[1]:
            raise ValueError(f"a sequence holds at most {self.page_table.shape[1] * self.page_size} positions, asked for {positions}")
        if need <= len(owned):
            return
        if need - len(owned) > len(self._free):
            raise MemoryError(f"{need - len(owned)} pages wanted, {len(self._free)} free")
        new = self._free[len(owned) - need:][::-1]
        # from pinned memory, which torch keeps until the copy is done: the host does not wait for what is queued
        ids = torch.tensor(new, dtype=torch.int32, pin_memory=self.page_table.is_cuda)
        self.page_table[seq, len(owned):need].copy_(ids, non_blocking=True)
        del self._free[len(owned) - need:]   # only now: what raised above has cost no page
        owned.extend(new)

    def release(self, seq: int) -> None:
        """Take all pages of sequence ``seq`` back."""
        self._check(seq)
        self.page_table[seq].fill_(-1)
        self._free.extend(reversed(self._owned[seq]))
        self._owned[seq] = []

    def layer(self, index: int, seqs: int | None = None) -> dict:
        """One layer's tensors, for the first ``seqs`` sequences or all, as keyword arguments of ``append`` and ``attention``."""
        scales = {} if self.k_scales is None else dict(k_scales=self.k_scales[index], v_scales=self.v_scales[index])
        return dict(k_pages=self.k[index], v_pages=self.v[index], page_table=self.page_table[:seqs], **scales)

    def describe(self) -> _lib.MkPagedModelCache:
        """The cache as ``mk_batched_set_paged_cache`` takes it."""
        layers, pages, heads, size, dim = self.k.shape
        scales = (None, None) if self.k_scales is None else (self.k_scales.data_ptr(), self.v_scales.data_ptr())
        first = _lib.MkPagedCache(self.k.data_ptr(), self.v.data_ptr(), *scales, heads * size * dim, size * dim, dim,
                                  _lib.MK_CACHE_BF16 if self.k_scales is None else _lib.MK_CACHE_E4M3, pages, size, heads, dim, 0)
        return _lib.MkPagedModelCache(first, pages * heads * size * dim, pages * heads, self.page_table.data_ptr(), self.page_table.shape[1],
                                      self.page_table.shape[0], self.page_table.shape[1])
