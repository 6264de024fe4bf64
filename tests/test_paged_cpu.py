"""Paged cache without a device: struct layouts, refusals of the C entry points and of the Python functions."""
import ctypes as C

import pytest
import torch

from thor_megakernels_b200 import _lib, paged


def good():
    """Structs that only a missing device can refuse (the pointers are never followed on the host)."""
    cache = _lib.MkPagedCache(4096, 8192, None, None, 2 * 16 * 64, 16 * 64, 64, _lib.MK_CACHE_BF16, 10, 16, 2, 64, 0)
    batch = _lib.MkPagedBatch(4096, 4, 4096, None, 4096, 3, 6, 4, 0)
    append = _lib.MkPagedAppend(4096, 4096, 4096, 4096, 4096, 4096, 512, 64, 512, 64, 512, 64, 8, 64, 100, 0)
    attention = _lib.MkPagedAttention(4096, 4096, 4096, 1 << 40, 512, 64, 8, 0.125)
    return cache, batch, append, attention


def test_struct_layouts_match():
    lib = _lib.load()
    for which, struct in enumerate((_lib.MkPagedCache, _lib.MkPagedBatch, _lib.MkPagedAppend, _lib.MkPagedAttention,
                                      _lib.MkPagedModelCache), start=4):
        assert lib.mk_abi_sizeof(which) == C.sizeof(struct), struct.__name__


CACHE = [dict(k_pages=None), dict(v_pages=8200), dict(format=2), dict(format=_lib.MK_CACHE_E4M3), dict(num_pages=0), dict(page_size=8),
         dict(page_size=48), dict(page_size=256), dict(num_kv_heads=0), dict(head_dim=80), dict(head_dim=256), dict(slot_stride=32),
         dict(slot_stride=66), dict(page_stride=0), dict(head_stride=-64), dict(page_stride=4095)]
BATCH = [dict(page_table=None), dict(positions=None), dict(error_word=None), dict(seqs=0), dict(tokens=0), dict(max_pages=0), dict(tokens=7),
         dict(table_stride=3), dict(seqs=_lib.MK_PAGED_MAX_SEQS + 1, cu_tokens=4096)]
APPEND = [dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(rope_sin=None), dict(rot_dim=8), dict(rot_dim=72), dict(rot_dim=80),
          dict(rope_positions=0), dict(k=4104), dict(k_token_stride=12), dict(num_q_heads=0), dict(rope_cos=4100)]
ATTENTION = [dict(q=None), dict(out=None), dict(num_q_heads=0), dict(num_q_heads=7), dict(q_token_stride=4), dict(scale=float("inf")),
             dict(scale=float("nan")), dict(out=4104)]


def changed(struct, changes):
    for name, value in changes.items():
        setattr(struct, name, value)


@pytest.mark.parametrize("which,changes", [(0, c) for c in CACHE] + [(1, c) for c in BATCH] + [(2, c) for c in APPEND])
def test_append_refuses(which, changes):
    lib = _lib.load()
    structs = good()
    changed(structs[which], changes)
    code = lib.mk_paged_append(structs[0], structs[1], structs[2], None)
    assert code in (_lib.MK_ERR_BAD_ARGUMENT, _lib.MK_ERR_UNSUPPORTED), changes
    assert lib.mk_last_error().startswith(b"mk_paged_append: ")


@pytest.mark.parametrize("which,changes", [(0, c) for c in CACHE] + [(1, c) for c in BATCH] + [(3, c) for c in ATTENTION])
def test_attention_refuses(which, changes):
    lib = _lib.load()
    structs = good()
    changed(structs[which], changes)
    code = lib.mk_paged_attention(structs[0], structs[1], structs[3], None)
    assert code in (_lib.MK_ERR_BAD_ARGUMENT, _lib.MK_ERR_UNSUPPORTED), changes
    assert lib.mk_last_error().startswith(b"mk_paged_attention: ")
    if which < 2:
        assert lib.mk_paged_attention_workspace(structs[0], structs[1], 8) == -1


def test_null_structs_are_refused():
    lib = _lib.load()
    cache, batch, append, attention = good()
    for args in ((None, batch, append), (cache, None, append), (cache, batch, None)):
        assert lib.mk_paged_append(*args, None) == _lib.MK_ERR_BAD_ARGUMENT
    for args in ((None, batch, attention), (cache, None, attention), (cache, batch, None)):
        assert lib.mk_paged_attention(*args, None) == _lib.MK_ERR_BAD_ARGUMENT
    assert lib.mk_paged_attention_workspace(None, None, 8) == -1


def test_cpu_tensors_are_refused():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    table, one = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.attention(rows, k, k, table, one)
    with pytest.raises(ValueError):
        paged.append(rows, rows, k, k, table, one)


def test_a_null_handle_gets_no_paged_cache():
    lib = _lib.load()
    assert lib.mk_batched_set_paged_cache(None, None) == _lib.MK_ERR_BAD_ARGUMENT
    assert b"null handle" in lib.mk_last_error()


def test_attention_refuses_what_its_workspace_cannot_describe():
    lib = _lib.load()
    cache, batch, _, attention = good()
    batch.seqs, batch.cu_tokens = 1025, 4096
    assert lib.mk_paged_attention(cache, batch, attention, None) == _lib.MK_ERR_UNSUPPORTED
    assert b"more sequences" in lib.mk_last_error()
    cache, batch, _, attention = good()
    cache.num_kv_heads = attention.num_q_heads = 0x8000
    assert lib.mk_paged_attention(cache, batch, attention, None) == _lib.MK_ERR_UNSUPPORTED
    assert b"KV heads" in lib.mk_last_error()


def test_the_first_call_on_a_device_is_not_captured(monkeypatch):
    monkeypatch.setattr(paged, "_error_words", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        paged._error_word(0)


def test_a_cache_needs_room_for_a_position():
    with pytest.raises(ValueError):
        paged.PagedKvCache(1, 4, 1, 64, max_positions=0, device="cpu")
