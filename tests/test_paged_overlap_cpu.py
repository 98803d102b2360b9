"""Accumulators whose rows share memory: written by several CTAs at once, so refused before any CUDA call."""
from __future__ import annotations

import pytest
import torch

import int4_b200
from int4_b200 import _lib

B, NKV, PAGE, WIDTH = 2, 2, 16, 3
SLOTS = PAGE * WIDTH


def _tensors():
    k = torch.zeros(6, NKV, PAGE, 64, dtype=torch.bfloat16)
    return k, torch.zeros_like(k), torch.zeros(B, WIDTH, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)


def _evict(weights, weights_out):
    k, v, table, lens = _tensors()
    return int4_b200.paged_evict(weights, lens, table, k, v, torch.zeros(B, 2, dtype=torch.int32), 32, weights_out=weights_out)


def _buffer():
    return torch.zeros(4 * B * NKV * SLOTS)


def _shared_rows():
    one = torch.zeros(B, NKV, SLOTS)
    return {"sequences": one[:1].expand(B, NKV, SLOTS), "heads": one[:, :1].expand(B, NKV, SLOTS),
            "half of the next head's": _buffer().as_strided((B, NKV, SLOTS), (NKV * SLOTS, SLOTS // 2, 1)),
            "the last word": _buffer().as_strided((B, NKV, SLOTS), (2 * SLOTS - 1, SLOTS, 1))}


@pytest.mark.parametrize("which", list(_shared_rows()))
def test_evict_refuses_an_output_whose_rows_share_memory(which):
    with pytest.raises(ValueError, match="weights_out.*same memory"):
        _evict(torch.zeros(B, NKV, SLOTS), _shared_rows()[which])


def test_evict_refuses_an_output_that_overlaps_its_weights():
    shape, strides = (B, NKV, SLOTS), (NKV * SLOTS, SLOTS, 1)
    buf = _buffer()
    w = buf.as_strided(shape, strides, 0)
    for out in (buf.as_strided(shape, strides, 1), buf.as_strided(shape, strides, NKV * SLOTS), buf.as_strided(shape, strides, B * NKV * SLOTS - 1),
                buf.as_strided(shape, (SLOTS, B * SLOTS, 1)), buf.as_strided(shape, (2 * NKV * SLOTS, SLOTS, 1)), w.flip(0)[1:2].expand(shape)):
        with pytest.raises(ValueError, match="weights_out.*same memory"):
            _evict(w, out)


def test_evict_takes_outputs_that_lie_apart_or_are_the_weights():
    shape = (B, NKV, SLOTS)
    buf = _buffer()
    w = buf.as_strided(shape, (NKV * SLOTS, SLOTS, 1))
    apart = [buf.as_strided(shape, (NKV * SLOTS, SLOTS, 1), B * NKV * SLOTS), w, buf.as_strided(shape, (NKV * SLOTS, SLOTS, 1)),
             torch.zeros(shape), torch.zeros(NKV, B, SLOTS).transpose(0, 1)]
    for out in apart:
        with pytest.raises(ValueError, match="GPU only|one device"):  # nothing else is wrong with them
            _evict(w, out)
    rows = torch.zeros(2, B, NKV, SLOTS).permute(1, 2, 0, 3)  # weights and outputs by turns
    with pytest.raises(ValueError, match="GPU only|one device"):
        _evict(rows[:, :, 0], rows[:, :, 1])


def test_c_evict_refuses_rows_that_overlap():
    L = _lib.lib()
    c = _lib.PAGED_CACHE.pack(0x1000, 0x2000, 2048, 1024, 64, 2048, 1024, 64, 0x3000, 3, 6, 2, 16, 64, 2, 3, 1)

    def evict(sb, sh):
        return L.i4b_paged_evict(c, 0x4000, 96, 48, 48, 0x5000, 0x5100, 2, 2, 32, 0, 0x6000, 0x6100, 0x6200, sb, sh, None)

    for sb, sh in ((96, 0), (0, 48), (96, 47), (47, 96), (-47, 96), (96, -1)):
        assert evict(sb, sh) == 4, (sb, sh)


def _attend(weights):
    k, v, table, lens = _tensors()
    return int4_b200.paged_decode_attention(torch.zeros(B, 4, 64, dtype=torch.bfloat16), k, v, table, lens, weights=weights)


@pytest.mark.parametrize("which", list(_shared_rows()))
def test_attention_refuses_weights_whose_rows_share_memory(which):
    with pytest.raises(ValueError, match="same memory"):
        _attend(_shared_rows()[which])


def test_attention_takes_weights_whose_rows_lie_apart():
    wide = torch.zeros(B, NKV, SLOTS + 40)
    slack = _buffer().as_strided((B, NKV, SLOTS + 8), (NKV * SLOTS, SLOTS, 1))  # rows as long as the tables' slots do not meet
    for w in (wide, wide[..., 3:], torch.zeros(NKV, B, SLOTS).transpose(0, 1), torch.zeros(SLOTS * 4).as_strided((B, NKV, SLOTS), (SLOTS, 2 * SLOTS, 1)), slack):
        with pytest.raises(ValueError, match="GPU only|one device"):
            _attend(w)


def test_c_attention_refuses_weights_that_overlap():
    L = _lib.lib()
    c = _lib.PAGED_CACHE.pack(0x1000, 0x2000, 2048, 1024, 64, 2048, 1024, 64, 0x3000, 3, 6, 2, 16, 64, 2, 3, 1)
    for sb, sh in ((96, 0), (0, 48), (96, 47), (47, 96)):
        assert L.i4b_paged_decode_attention(c, 0x4000, 512, 64, 8, 0x5000, 0.125, 0x6000, 0x8000, sb, sh, 0x7000, 1 << 40, None) == 4
