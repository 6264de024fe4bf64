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
