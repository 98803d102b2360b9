"""The page bookkeeping of PagedKVCache on the CPU (no kernel runs)."""
from __future__ import annotations

import pytest
import torch

from int4_b200 import PagedKVCache
from int4_b200._lib import Int4B200Error


def _cache(**kw):
    d = dict(num_pages=6, max_seqs=3, max_len=40, page_size=8, device=torch.device("cpu"))
    return PagedKVCache(2, 2, 64, **{**d, **kw})


def test_reserve_is_all_or_nothing():
    c = _cache()
    c.reserve({0: 9, 2: 8})
    assert [len(p) for p in c.pages] == [2, 0, 1] and len(c.free_pages) == 3
    assert c.table[0].tolist()[:3] == [*c.pages[0], -1] and c.table[2, 0].item() == c.pages[2][0]
    c.lengths[0], c.lengths[2] = 9, 8
    c.reserve({0: 7})  # within the second page
    assert len(c.pages[0]) == 2
    with pytest.raises(Int4B200Error, match="4 pages wanted, 3 free"):
        c.reserve({1: 17, 2: 1})
    with pytest.raises(Int4B200Error, match="41 slots of 40"):
        c.reserve({1: 1, 0: 32})
    assert len(c.free_pages) == 3 and c.pages[1] == []
    with pytest.raises(ValueError, match="sequence 3"):
        c.reserve({3: 1})


def test_steps_take_a_page_when_one_is_full_and_free_gives_all_back():
    c = _cache()
    c.reserve({1: 7})
    c.lengths[1] = 7
    for n, pages in ((8, 1), (9, 2), (10, 2)):
        c.reserve_step()
        assert c.lengths == [0, n, 0] and len(c.pages[1]) == pages
    c.free(1)
    assert sorted(c.free_pages) == list(range(6)) and (c.table == -1).all() and c.lengths == [0, 0, 0]


@pytest.mark.parametrize("kw, words", [(dict(page_size=12), "page size"), (dict(max_seqs=4097), "max_seqs"), (dict(dtype=torch.float32), "bfloat16"),
                                       (dict(num_pages=0), "num_pages"), (dict(max_len=400000, track_weights=True), "max_len")])
def test_refusals(kw, words):
    with pytest.raises(ValueError, match=words):
        _cache(**kw)
    with pytest.raises(ValueError, match="track_weights"):
        _cache().evict(8)
    with pytest.raises(ValueError, match="budget"):
        _cache(track_weights=True).evict(8, recent=9)
