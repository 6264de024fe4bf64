"""PagedKvCache's handing out of pages, without a device."""
import pytest
import torch

from thor_megakernels_b200 import paged


def cache(**kw):
    return paged.PagedKvCache(1, 8, 1, 64, page_size=16, max_seqs=3, max_positions=64, device="cpu", **kw)


@pytest.mark.parametrize("seq", [-1, -3, 3, 100])
def test_sequences_that_are_not_there_are_refused(seq):
    c = cache()
    c.reserve(2, 20)
    before = c.page_table.clone()
    with pytest.raises(IndexError):
        c.reserve(seq, 40)
    with pytest.raises(IndexError):
        c.release(seq)
    assert c.free_pages == 6 and torch.equal(c.page_table, before)


def test_a_reserve_that_fails_costs_no_page(monkeypatch):
    c = cache()
    c.reserve(0, 20)
    table = c.page_table.clone()

    def fails(*args, **kw):
        raise RuntimeError("no memory")

    with monkeypatch.context() as m:
        m.setattr(torch, "tensor", fails)
        with pytest.raises(RuntimeError, match="no memory"):
            c.reserve(1, 50)
    assert c.free_pages == 6 and torch.equal(c.page_table, table)
    c.reserve(1, 50)
    assert c.free_pages == 2 and c.page_table[1].tolist() == [2, 3, 4, 5]


def test_pages_are_handed_out_in_order_and_taken_back():
    c = cache()
    c.reserve(0, 17)
    c.reserve(1, 1)
    c.reserve(0, 33)
    assert c.page_table.tolist() == [[0, 1, 3, -1], [2, -1, -1, -1], [-1] * 4]
    c.release(0)
    assert c.free_pages == 7 and c.page_table[0].tolist() == [-1] * 4
    c.reserve(2, 64)
    assert c.page_table[2].tolist() == [0, 1, 3, 4]
    with pytest.raises(MemoryError):
        c.reserve(0, 64)
    assert c.free_pages == 3


def test_append_refuses_keys_and_values_in_the_same_pages():
    """Both would be written by blocks of their own, in any order."""
    from test_paged_cpu import good

    from thor_megakernels_b200 import _lib

    lib = _lib.load()
    for changes in (dict(v_pages=4096), dict(format=_lib.MK_CACHE_E4M3, k_scales=4096, v_scales=4096)):
        cache, batch, append, _ = good()
        for name, value in changes.items():
            setattr(cache, name, value)
        assert lib.mk_paged_append(cache, batch, append, None) == _lib.MK_ERR_BAD_ARGUMENT
        assert b"of their own" in lib.mk_last_error()


@pytest.mark.parametrize("value,code", [(1, "MK_ERR_DEVICE_WAIT"), (2, "MK_ERR_BAD_ARGUMENT"), (0, None)])
def test_an_error_is_wiped_out_before_the_next_call_can_report(monkeypatch, value, code):
    from thor_megakernels_b200 import _lib

    log = []

    class Word:
        def item(self):
            log.append("read")
            return value

        def zero_(self):
            log.append("zero")

    monkeypatch.setattr(paged, "_error_word", lambda device: Word())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: log.append("sync"))
    if code is None:
        paged.check_errors("cuda:0")
        assert log == ["sync", "read"]
        return
    with pytest.raises(_lib.MegakernelError) as raised:
        paged.check_errors("cuda:0")
    assert raised.value.code == getattr(_lib, code)
    assert log == ["sync", "read", "zero", "sync"]
