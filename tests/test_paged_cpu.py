"""What the paged-cache operators and token_logprobs refuse, before any CUDA call: no GPU needed."""
from __future__ import annotations

import pytest
import torch

import int4_b200
from int4_b200 import _lib


def _step(B=2, nq=8, nkv=2, dim=64, page=16, pages=6, width=3, dtype=torch.bfloat16):
    k = torch.zeros(pages, nkv, page, dim, dtype=dtype)
    return {"k": k, "v": torch.zeros_like(k), "q": torch.zeros(B, nq, dim, dtype=dtype),
            "table": torch.zeros(B, width, dtype=torch.int32), "lens": torch.zeros(B, dtype=torch.int32),
            "weights": torch.zeros(B, nkv, width * page)}


def _attend(s, **kw):
    return int4_b200.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], **kw)


@pytest.mark.parametrize("change, words", [
    (dict(k=torch.zeros(6, 2, 16, 64)), "bfloat16"),
    (dict(k=torch.zeros(6, 2, 12, 64, dtype=torch.bfloat16), v=torch.zeros(6, 2, 12, 64, dtype=torch.bfloat16)), "page size"),
    (dict(k=torch.zeros(6, 2, 16, 96, dtype=torch.bfloat16), v=torch.zeros(6, 2, 16, 96, dtype=torch.bfloat16)), "head_dim"),
    (dict(v=torch.zeros(6, 2, 16, 128, dtype=torch.bfloat16)), "k_cache and v_cache"),
    (dict(v=torch.zeros(6, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3)), "unit stride"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "block_table"),
    (dict(table=torch.zeros(3, 2, dtype=torch.int32).T), "block_table"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "lens"),
    (dict(q=torch.zeros(2, 7, 64, dtype=torch.bfloat16)), "query heads"),
    (dict(q=torch.zeros(2, 8, 64, dtype=torch.float16)), "q must be"),
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "q must be"),
    ({}, "GPU only"),
])
def test_attention_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        _attend({**_step(), **change})


def test_attention_refuses_weights_and_out_of_other_shapes():
    s = _step()
    for w in (s["weights"][:, :, :-1], s["weights"][:, :1], s["weights"].double(), s["weights"].transpose(1, 2)):
        with pytest.raises(ValueError, match="weights"):
            _attend(s, weights=w)
    with pytest.raises(ValueError, match="same memory"):
        _attend(s, weights=s["weights"][:1].expand(2, 2, 48))
    for out in (torch.zeros(2, 8, 64), torch.zeros(2, 8, 128, dtype=torch.bfloat16)[..., :64]):
        with pytest.raises(ValueError, match="out must be"):
            _attend(s, out=out)


def test_append_refuses():
    s = _step()
    T = 2
    good = dict(qkv=torch.zeros(T, 12 * 64, dtype=torch.bfloat16), cos=torch.zeros(32, 64), sin=torch.zeros(32, 64),
                positions=torch.zeros(T, dtype=torch.int32), slots=torch.zeros(T, dtype=torch.int32), block_table=s["table"],
                k_cache=s["k"], v_cache=s["v"])
    for change, words in ((dict(qkv=torch.zeros(T, 12 * 64)), "qkv"), (dict(qkv=torch.zeros(T, 4 * 64, dtype=torch.bfloat16)), "queries"),
                          (dict(qkv=torch.zeros(T, 700, dtype=torch.bfloat16)), "queries"),
                          (dict(cos=torch.zeros(32, 64, dtype=torch.float16), sin=torch.zeros(32, 64, dtype=torch.float16)), "cos and sin"),
                          (dict(cos=torch.zeros(31, 64)), "cos and sin"), (dict(slots=torch.zeros(T)), "slots"),
                          (dict(positions=torch.zeros(1, dtype=torch.int32)), "positions"),
                          (dict(seqs=torch.zeros(T, dtype=torch.int64)), "seqs"),
                          (dict(block_table=s["table"][:1]), "without seqs"), ({}, "GPU only")):
        with pytest.raises(ValueError, match=words):
            int4_b200.paged_kv_append(**{**good, **change})


def test_evict_refuses():
    s = _step()
    new = torch.zeros(2, 2, dtype=torch.int32)

    def call(budget=32, recent=0, table=new, weights=s["weights"], **kw):
        return int4_b200.paged_evict(weights, s["lens"], s["table"], s["k"], s["v"], table, budget, recent=recent, **kw)

    for kw, words in ((dict(budget=0), "budget"), (dict(recent=33), "recent"), (dict(recent=-1), "recent"), (dict(budget=33), "new_table"),
                      (dict(table=new[:1]), "new_table"), (dict(weights=s["weights"][..., 1:]), "weights"),
                      (dict(weights_out=torch.zeros(2, 2, 47)), "weights_out"), ({}, "GPU|one device")):
        with pytest.raises(ValueError, match=words):
            call(**kw)


def test_logprobs_refuses():
    z, t = torch.zeros(3, 40), torch.zeros(3, dtype=torch.int64)
    for args, words in (((z.double(), t), "logits"), ((z, t.int()), "targets"), ((z, t[:2]), "targets"), ((z, t, 33), "alternatives"),
                        ((z, t, -1), "alternatives"), ((z[:, :4], t, 5), "alternatives"), ((z[:, :0], t), "logits"), ((z, t), "GPU only")):
        with pytest.raises(ValueError, match=words):
            int4_b200.token_logprobs(*args)


# ---- the C entries, with pointers that are never followed


def _struct(**kw):
    d = dict(k=0x1000, v=0x2000, k_stride_page=2048, k_stride_head=1024, k_stride_token=64, v_stride_page=2048, v_stride_head=1024,
             v_stride_token=64, block_table=0x3000, table_stride=3, num_pages=6, kv_heads=2, page_size=16, head_dim=64, seqs=2,
             max_pages=3, dtype=1)
    d = {**d, **kw}
    return _lib.PAGED_CACHE.pack(*(0 if x is None else x for x in d.values()))


def _c_attend(cache, nq=8, q=0x4000, weights=None, ws=0x7000, size=1 << 40):
    return _lib.lib().i4b_paged_decode_attention(cache, q, nq * 64, 64, nq, 0x5000, 0.125, 0x6000, weights, 96, 48, ws, size, None)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=2), 1), (dict(k=None), 1), (dict(block_table=None), 1), (dict(head_dim=80), 2), (dict(page_size=12), 2),
    (dict(page_size=0), 2), (dict(num_pages=0), 2), (dict(num_pages=1 << 32), 2), (dict(seqs=4097), 2), (dict(seqs=-1), 2),
    (dict(max_pages=1 << 27), 2), (dict(max_pages=-1), 2), (dict(kv_heads=0), 2), (dict(k=0x1008), 4), (dict(v_stride_token=68), 4),
    (dict(k_stride_page=-2048), 4), (dict(seqs=4096, max_pages=1 << 26), 2)])
def test_c_attention_statuses(change, status):
    assert _c_attend(_struct(**change)) == status


def test_c_statuses_of_the_other_arguments():
    L = _lib.lib()
    assert _c_attend(_struct(kv_heads=1), nq=1025) == 2  # query heads per kv head
    assert _c_attend(_struct(), nq=7) == 2 and _c_attend(_struct(), q=None) == 1 and _c_attend(_struct(), q=0x4008) == 4
    assert _c_attend(_struct(seqs=0)) == 0  # nothing to do
    assert _c_attend(_struct(kv_heads=1, k_stride_head=3, v_stride_head=5), q=None) == 1  # a stride that is never used
    assert L.i4b_paged_decode_attention(None, 0, 0, 0, 8, 0, 1.0, 0, None, 0, 0, 0, 0, None) == 1
    c = _struct()

    def append(tokens=2, nq=8, table_dtype=2, max_pos=32, qkv=0x4000, stride=768, cos=0x8000):
        return L.i4b_paged_kv_append(c, qkv, stride, tokens, nq, cos, 0x9000, table_dtype, max_pos, 0x5000, 0x5100, None, 0x6000, None)

    assert append(table_dtype=0) == 1 and append(tokens=-1) == 2 and append(nq=0) == 2 and append(max_pos=0) == 2
    assert append(qkv=None) == 1 and append(stride=770) == 4 and append(cos=0x8004) == 4 and append(tokens=0) == 0

    def evict(width=48, new_pages=2, budget=32, recent=0, weights=0x4000):
        return L.i4b_paged_evict(c, weights, 96, 48, width, 0x5000, 0x5100, 2, new_pages, budget, recent, 0x6000, 0x6100,
                                 0x6200, 96, 48, None)

    assert evict(width=47) == 2 and evict(width=(1 << 30) + 1) == 2 and evict(budget=(1 << 30) + 1, new_pages=1 << 30) == 2
    assert evict(new_pages=1) == 2 and evict(budget=0) == 2 and evict(recent=33) == 2 and evict(weights=None) == 1

    def logprobs(dtype=1, rows=2, n=100, stride=100, top=0, x=0x4000, ids=None):
        return L.i4b_token_logprobs(x, dtype, rows, n, stride, 0x5000, top, 0x6000, 0x6100, 0x6200, ids, None)

    assert logprobs(dtype=3) == 1 and logprobs(n=(1 << 30) + 1) == 2 and logprobs(n=0) == 2 and logprobs(top=33) == 2 and logprobs(n=4, top=5) == 2 and logprobs(rows=-1) == 2
    assert logprobs(x=None) == 1 and logprobs(top=3) == 1 and logprobs(x=0x4001) == 4 and logprobs(rows=0) == 0


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 72, 128, 1000, 4096])
def test_division_by_the_page_size(page):
    """The kernels divide a slot by the page size with a multiplication: the same constants, checked in whole numbers."""
    shift = max(1, (page - 1).bit_length())
    mul = ((1 << (31 + shift)) + page - 1) // page
    assert mul < 1 << 32
    for n in [0, 1, page - 1, page, page + 1, 12345, (1 << 31) - 65] + [m * page + d for m in (7, 1000003, ((1 << 31) - 65) // page) for d in (-1, 0)]:
        assert (n * mul >> 32) >> (shift - 1) == n // page, (n, page)
