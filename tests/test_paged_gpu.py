"""The paged-cache operators against plain 64-bit implementations, at the sizes and masks where they can go wrong.

Tolerances: ``half`` is half a step of the type (finfo.eps / 2).  The attention rounds each probability and the output
once, so an output is within half * (sum p |v| + |out|), plus what the fp32 arithmetic of scores and sums adds:
``_fp32`` bounds the relative error of a probability.  Caches are filled with NaN wherever no sequence has written.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _cache(pages, nkv, page, dim, dtype, layout, gen, fill=math.nan):
    shape = (pages, nkv, page, dim) if layout == "heads" else (pages, page, nkv, dim)
    x = torch.full(shape, fill, device="cuda", dtype=dtype)
    return x.transpose(1, 2) if layout == "tokens" else x


def _filled(lens, nq, nkv, dim, page, dtype=torch.bfloat16, layout="heads", seed=0, spare=2, width=None):
    """Queries, a cache that holds sequences of ``lens``, and its block table (pages in random order)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    pages = sum(need) + spare
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), width), -7, device="cuda", dtype=torch.int32)
    k, v = (_cache(pages, nkv, page, dim, dtype, layout, gen) for _ in "kv")
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        for i in range(need[b]):
            m, p = min(page, n - i * page), order[at + i].long()
            k[p, :, :m] = torch.randn(nkv, m, dim, device="cuda", generator=gen).to(dtype)
            v[p, :, :m] = torch.randn(nkv, m, dim, device="cuda", generator=gen).to(dtype)
        at += need[b]
    q = (1.5 * torch.randn(len(lens), nq, dim, device="cuda", generator=gen)).to(dtype)
    return q, k, v, table, torch.tensor(lens, device="cuda", dtype=torch.int32)


def _reference(q, k, v, table, lens, scale=None):
    """(out, sum p |v|, weights, bound of a probability's relative fp32 error), in 64 bits, from the definition."""
    B, nq, dim = q.shape
    nkv, page = k.shape[1:3]
    G, cap = nq // nkv, table.shape[1] * page
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(B, nq, dim, device="cuda", dtype=torch.float64)
    mag, weights, worst = torch.zeros_like(out), torch.zeros(B, nkv, cap, device="cuda", dtype=torch.float64), 0.0
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        entries = table[b, torch.arange(n, device="cuda") // page].long()
        slots = torch.arange(n, device="cuda")
        ok = (entries >= 0) & (entries < k.shape[0])
        slots, entries = slots[ok], entries[ok]
        if not len(slots):
            continue
        kk, vv = k[entries, :, slots % page].double(), v[entries, :, slots % page].double()
        for h in range(nq):
            qd = q[b, h].double()
            s = kk[:, h // G] @ qd * scale
            p = torch.softmax(s, 0)
            out[b, h], mag[b, h] = p @ vv[:, h // G], p @ vv[:, h // G].abs()
            weights[b, h // G, slots] += p
            # a score: dim products and sums, the scale, the subtraction of the maximum, all in fp32
            worst = max(worst, float((kk[:, h // G].abs() @ qd.abs()).max()) * abs(scale))
    return out, mag, weights, (dim + 8) * 2 ** -24 * worst * 2 + 2 ** -20


def _check(q, k, v, table, lens, weights=False, scale=None, **kw):
    import int4_b200

    ref, mag, wref, eps = _reference(q, k, v, table, lens, scale)
    w = None
    if weights:
        gen = torch.Generator(device="cuda").manual_seed(5)
        w0 = torch.rand(wref.shape[0], wref.shape[1], wref.shape[2] + 3, device="cuda", generator=gen)
        w = w0.clone()
    out = int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w, scale=scale, **kw)
    half = _half(q.dtype)
    tiny = torch.finfo(q.dtype).smallest_normal
    tol = (half * (1 + half) + 2 * eps) * (mag + ref.abs()) + tiny
    bad = ((out.double() - ref).abs() > tol) | ~torch.isfinite(out)
    assert not bad.any(), (int(bad.sum()), float((out.double() - ref).abs().max()))
    if weights:
        want = w0.double()
        want[..., :wref.shape[2]] += wref
        G = q.shape[1] // k.shape[1]
        tol = torch.full_like(want, 0.0)
        tol[..., :wref.shape[2]] = wref * (2 * eps + G * 2 ** -23) + 2 ** -23 * want[..., :wref.shape[2]]
        tol = torch.where(want == w0.double(), 0.0, tol)  # slots that hold nothing are left as they were
        assert ((w.double() - want).abs() <= tol).all(), float((w.double() - want).abs().max())
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(4, 1), (8, 8), (14, 2), (16, 2), (16, 1), (34, 2)])
def test_attention_of_ragged_lengths(cuda_device, dtype, dim, nq, nkv):
    _check(*_filled([0, 1, 31, 32, 33, 137, 64, 500], nq, nkv, dim, 16, dtype, seed=nq + dim), weights=True)


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_attention_pages_and_layouts(cuda_device, page, layout):
    _check(*_filled([7, 8, 9, 300, 0, 1023], 8, 2, 64, page, layout=layout, seed=page), weights=True)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [65], [20000], [3] * 300, [1000] + [0] * 50 + [1]])
def test_attention_few_and_many_sequences(cuda_device, lens):
    _check(*_filled(lens, 8, 2, 64, 32, seed=len(lens)), weights=len(lens) < 100)


def test_attention_of_long_sequences_split_and_joined(cuda_device):
    _check(*_filled([50001, 3, 70000], 8, 2, 64, 128, torch.float16, seed=1), weights=True)
    _check(*_filled([40000], 4, 1, 128, 64, seed=2))


def test_attention_scale_and_large_scores(cuda_device):
    q, k, v, table, lens = _filled([200, 77], 8, 2, 64, 16, torch.float16, seed=3)
    _check(q, k, v, table, lens, scale=0.37)
    _check(q * 16, k, v, table, lens, weights=True)  # scores of +-100: nearly one-hot rows
    _check(q, k, v, table, lens, scale=0.0, weights=True)


def test_attention_leaves_out_pages_outside_the_cache(cuda_device):
    q, k, v, table, lens = _filled([200, 40, 64], 8, 2, 64, 16, seed=4)
    table[0, 3] = -1
    table[0, 7] = k.shape[0]
    table[1, :] = 2 ** 31 - 1  # a sequence without any page: an empty row
    out = _check(q, k, v, table, lens, weights=True)
    assert (out[1] == 0).all()


def test_attention_clamps_lengths_to_the_table(cuda_device):
    q, k, v, table, lens = _filled([48, 48, 48], 8, 2, 64, 16, seed=5)
    _check(q, k, v, table, torch.tensor([49, 2 ** 31 - 1, -5], device="cuda", dtype=torch.int32), weights=True)


def test_attention_infinities_and_nan_stay_in_their_rows(cuda_device):
    import int4_b200

    q, k, v, table, lens = _filled([40, 40, 40], 8, 2, 64, 16, seed=6)
    want = int4_b200.paged_decode_attention(q, k, v, table, lens)
    k[table[1, 1].long(), 0, 3] = math.inf  # within sequence 1's length, kv head 0: a score of +-inf or NaN
    v[table[2, 1].long(), 1, 3] = math.nan
    out = int4_b200.paged_decode_attention(q, k, v, table, lens)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1, 4:], want[1, 4:]) and torch.equal(out[2, :4], want[2, :4])
    assert torch.isnan(out[2, 4:]).all()


def test_attention_strided_queries_and_given_output(cuda_device):
    q, k, v, table, lens = _filled([90, 17], 8, 2, 64, 16, seed=7)
    wide = torch.zeros(2, 3, 8, 72, device="cuda", dtype=q.dtype)
    wide[:, 1, :, :64] = q
    out = torch.empty(2, 8, 64, device="cuda", dtype=q.dtype)
    assert _check(wide[:, 1, :, :64], k, v, table, lens, out=out) is out
    odd = torch.zeros(2, 8, 67, device="cuda", dtype=q.dtype)[..., 3:]  # rows that no 16-byte load can start
    odd.copy_(q)
    _check(odd, k, v, table, lens)
    _check(q, k, v, torch.cat([table, table], 1)[:, :table.shape[1]], lens, weights=True)  # rows of a wider table
    one = _filled([70], 4, 1, 64, 16, seed=8)
    _check(one[0].as_strided((1, 4, 64), (3, 64, 1)), *one[1:])  # a stride of a dimension of one
    flat = torch.zeros(4 * 64 + 3, device="cuda", dtype=q.dtype)[3:].view(1, 4, 64)  # contiguous, and misaligned
    _check(flat.copy_(one[0]), *one[1:])


def test_attention_without_table_columns_or_sequences(cuda_device):
    import int4_b200

    q, k, v, table, lens = _filled([5, 6], 8, 2, 64, 16, seed=9)
    assert (int4_b200.paged_decode_attention(q, k, v, table[:, :0], lens, weights=torch.empty(2, 2, 0, device="cuda")) == 0).all()
    assert int4_b200.paged_decode_attention(q[:0], k, v, table[:0], lens[:0]).shape == (0, 8, 64)


def test_attention_repeats_bit_by_bit_and_on_another_stream(cuda_device):
    import int4_b200

    q, k, v, table, lens = _filled([5000, 33, 2100], 8, 2, 64, 16, seed=10)
    a = int4_b200.paged_decode_attention(q, k, v, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = [int4_b200.paged_decode_attention(q, k, v, table, lens) for _ in range(4)]
    c = [int4_b200.paged_decode_attention(q, k, v, table, lens) for _ in range(4)]  # both streams at once
    torch.cuda.synchronize()
    assert all(torch.equal(a, x) for x in b + c)


def test_attention_captured_twice_and_replayed_together(cuda_device):
    """Two graphs of different lengths, replayed at once on two streams: neither uses the other's workspace."""
    import int4_b200

    sets, graphs = [], []
    for i in range(2):
        q, k, v, table, lens = _filled([4000 + i, 100], 8, 2, 64, 16, seed=11 + i)
        w = torch.zeros(2, 2, table.shape[1] * 16, device="cuda")
        out = torch.empty_like(q)
        int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w, out=out)
        graphs.append(g)
        sets.append((q, k, v, table, lens, w, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in (3900, 64, 0):  # lengths change between replays
        for i in range(2):
            sets[i][4].fill_(n)
            sets[i][5].zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for q, k, v, table, lens, w, out in sets:
            short = torch.tensor([n, min(n, 100)], device="cuda", dtype=torch.int32)
            ref, mag, wref, eps = _reference(q, k, v, table, short)
            tol = (_half(q.dtype) * 1.01 + 2 * eps) * (mag + ref.abs()) + 1e-30
            assert ((out[0].double() - ref[0]).abs() <= tol[0]).all()
            assert ((w[0].double() - 5 * wref[0]).abs() <= 5 * wref[0] * (2 * eps + 2 ** -19) + 1e-30).all()


def test_attention_offsets_beyond_32_bits(cuda_device):
    """A cache of more than 2^31 elements: the last pages are the ones in use."""
    nkv, page, dim = 8, 64, 64
    pages = (1 << 31) // (nkv * page * dim) + 200
    q, k0, v0, t0, lens = _filled([300, 64], 16, nkv, dim, page, seed=13, spare=0)
    k = torch.empty(pages, nkv, page, dim, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    n = k0.shape[0]
    k[-n:], v[-n:] = k0, v0
    table = torch.where(t0 >= 0, t0 + (pages - n), t0)
    _check(q, k, v, table, lens, weights=True)


# ------------------------------------------------------------------ append


def _rope64(x, cos, sin):
    x, half = x.double(), x.shape[-1] // 2
    return x * cos.double() + torch.cat([-x[..., half:], x[..., :half]], -1) * sin.double(), \
        x.abs() * cos.double().abs() + torch.cat([x[..., half:], x[..., :half]], -1).abs() * sin.double().abs()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("table32", [False, True])
@pytest.mark.parametrize("nq,nkv,dim,page,layout,T", [(8, 2, 64, 16, "heads", 1), (7, 7, 128, 24, "tokens", 50), (40, 5, 64, 8, "tokens", 33),
                                                       (64, 8, 128, 64, "heads", 5)])
def test_append_rotates_and_writes(cuda_device, dtype, table32, nq, nkv, dim, page, layout, T):
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(T)
    B, width, max_pos = 5, 6, 400
    pages = B * width + 3
    k, v = (_cache(pages, nkv, page, dim, dtype, layout, gen, 0.5) for _ in "kv")
    table = torch.randperm(pages, device="cuda", generator=gen)[:B * width].to(torch.int32).view(B, width)
    ang = 10 * torch.rand(max_pos, dim, device="cuda", generator=gen)
    tdt = torch.float32 if table32 else dtype
    cos, sin = ang.cos().to(tdt), ang.sin().to(tdt)
    qkv = torch.randn(T, (nq + 2 * nkv) * dim + 8, device="cuda", generator=gen).to(dtype)[:, 8:]
    places = torch.randperm(B * width * page, device="cuda", generator=gen)[:T]  # distinct (sequence, slot)
    seqs, slots = (places // (width * page)).to(torch.int32), (places % (width * page)).to(torch.int32)
    pos = torch.randint(0, max_pos, (T,), device="cuda", generator=gen).to(torch.int32)
    k0, v0 = k.clone(), v.clone()
    q = int4_b200.paged_kv_append(qkv, cos, sin, pos, slots, table, k, v, seqs=seqs)
    x = qkv.reshape(T, nq + 2 * nkv, dim)
    ref, mag = _rope64(x, cos[pos.long()][:, None], sin[pos.long()][:, None])
    tol = _half(dtype) * ref.abs() + 4 * 2 ** -24 * mag + torch.finfo(dtype).smallest_normal * _half(dtype)
    assert ((q.double() - ref[:, :nq]).abs() <= tol[:, :nq]).all()
    page_at = table[seqs.long(), (slots // page).long()].long()
    got = k[page_at, :, (slots % page).long()]
    assert ((got.double() - ref[:, nq:nq + nkv]).abs() <= tol[:, nq:nq + nkv]).all()
    assert torch.equal(v[page_at, :, (slots % page).long()], x[:, nq + nkv:])
    k0[page_at, :, (slots % page).long()] = got  # everything else is left as it was
    v0[page_at, :, (slots % page).long()] = x[:, nq + nkv:]
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_append_padding_writes_nothing(cuda_device):
    import int4_b200

    k = torch.full((4, 2, 16, 64), 0.5, device="cuda", dtype=torch.bfloat16)
    v = k.clone()
    table = torch.tensor([[0, 1], [2, -1]], device="cuda", dtype=torch.int32)
    cos = torch.ones(10, 64, device="cuda")
    sin = torch.zeros(10, 64, device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    #            below the slots, above, no page, no such sequences, positions outside
    slots = torch.tensor([-1, 32, 20, 3, 3, 4, 5], **i32)
    seqs = torch.tensor([0, 0, 1, -1, 2, 0, 0], **i32)
    pos = torch.tensor([1, 1, 1, 1, 1, -1, 10], **i32)
    qkv = torch.ones(7, 8 * 64, device="cuda", dtype=torch.bfloat16)
    q = int4_b200.paged_kv_append(qkv, cos, sin, pos, slots, table, k, v, seqs=seqs)
    assert (k == 0.5).all() and (v == 0.5).all()
    assert (q[:5] == 1).all() and (q[5:] == 0).all()
    # without seqs: token i is sequence i's
    int4_b200.paged_kv_append(qkv[:2], cos, sin, pos[:2], torch.tensor([17, 2], **i32), table, k, v)
    assert (k[1, :, 1] == 1).all() and (k[2, :, 2] == 1).all() and (k == 1).sum() == 2 * 2 * 64
    assert int4_b200.paged_kv_append(qkv[:0], cos, sin, pos[:0], pos[:0], table, k, v).shape == (0, 4, 64)


# ------------------------------------------------------------------ eviction


def _evict_reference(w, lens, budget, recent):
    B, nkv, W = w.shape
    kept = torch.full((B, nkv, budget), -1, dtype=torch.int32)
    w = w.cpu()
    for b in range(B):
        n = int(lens[b])
        for h in range(nkv):
            idx = list(range(n))
            if n > budget:
                old = n - recent
                row = [(-math.inf if math.isnan(x) else x, not math.isnan(x)) for x in w[b, h, :old].tolist()]
                best = sorted(range(old), key=lambda i: (-row[i][0], not row[i][1], i))[:budget - recent]
                idx = sorted(best) + list(range(old, n))
            kept[b, h, :len(idx)] = torch.tensor(idx, dtype=torch.int32)
    return kept


def _run_evict(w, lens, page, budget, recent, nkv, dim=64, dtype=torch.bfloat16, layout="heads", seed=0, in_place=False):
    import int4_b200

    _, k, v, table, dlens = _filled(lens, nkv, nkv, dim, page, dtype, layout, seed, spare=0, width=-(-w.shape[2] // page))
    used, new_w = k.shape[0], -(-budget // page)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = (used + torch.randperm(len(lens) * new_w, device="cuda", generator=gen)).to(torch.int32).view(len(lens), new_w)
    big = [_cache(used + len(lens) * new_w, nkv, page, dim, dtype, layout, gen, 0.25) for _ in "kv"]
    for x, y in zip(big, (k, v)):
        x[:used] = y
    w0 = w.clone()
    new_lens, kept, wo = int4_b200.paged_evict(w, dlens, table, big[0], big[1], new, budget, recent=recent,
                                               weights_out=w if in_place else None)
    want = _evict_reference(w0, lens, budget, recent).cuda()
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    assert torch.equal(kept, want)
    assert (wo.data_ptr() == w.data_ptr()) == in_place
    for b, n in enumerate(lens):
        m = min(n, budget)
        at = torch.arange(m, device="cuda")
        for h in range(nkv):
            idx = want[b, h, :m].long()
            assert torch.equal(wo[b, h, :m].view(torch.int32), w0[b, h, idx].view(torch.int32)) and (wo[b, h, m:] == 0).all()
            for x in big:
                rows = x[new[b].long()[at // page], h, at % page]
                assert torch.equal(rows, x[table[b].long()[idx // page], h, idx % page])
        for x in big:  # rows behind the last kept one are left as they were
            for i in range(m, new_w * page):
                assert (x[new[b, i // page].long(), :, i % page] == 0.25).all()
    for x, y in zip(big, (k, v)):
        assert torch.equal(x[:used].view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (64, 0), (100, 37), (100, 100), (33, 32), (513, 5)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_keeps_the_heaviest_and_the_recent(cuda_device, budget, recent, in_place):
    gen = torch.Generator(device="cuda").manual_seed(budget)
    lens = [0, 1, 700, 64, 100, 101, 2000]
    w = torch.rand(len(lens), 2, 2000, device="cuda", generator=gen)
    w = torch.where(w < 0.3, 0.0, torch.where(w < 0.5, 0.25, w))  # ties among the kept and the dropped
    _run_evict(w, lens, 16, budget, recent, 2, seed=budget + recent, in_place=in_place)


@pytest.mark.parametrize("dim,page,dtype,layout", [(128, 24, torch.float16, "tokens"), (64, 64, torch.bfloat16, "tokens"), (128, 8, torch.bfloat16, "heads")])
def test_evict_layouts(cuda_device, dim, page, dtype, layout):
    gen = torch.Generator(device="cuda").manual_seed(page)
    _run_evict(torch.rand(3, 5, 384, device="cuda", generator=gen), [312, 200, 311], page, 130, 9, 5, dim, dtype, layout)


def test_evict_orders_every_float(cuda_device):
    special = [math.inf, -math.inf, math.nan, 0.0, -0.0, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0, 1.0, -math.nan, -1.0, 0.0, -0.0, math.inf]
    w = torch.tensor(special, device="cuda").repeat(1, 2, 6)
    for budget in (1, 12, 40, 70, 95):
        _run_evict(w.clone(), [96], 16, budget, 0, 2, seed=budget)
    _run_evict(torch.full((1, 2, 96), math.nan, device="cuda"), [96], 16, 40, 3, 2)
    _run_evict(torch.zeros(1, 2, 96, device="cuda"), [96], 16, 40, 3, 2)  # nothing was ever attended: the first and the recent


def test_evict_long_rows(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = torch.rand(1, 2, 70016, device="cuda", generator=gen) ** 8
    w[0, 1, 1000:60000] = 0.0  # long runs of one value
    _run_evict(w, [70003], 64, 3000, 100, 2)


def test_steps_of_a_run_with_eviction(cuda_device):
    """Append, attend with weights, evict into new pages, go on: the same as attention over the kept rows."""
    import int4_b200

    B, nq, nkv, dim, page = 3, 8, 2, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(20)
    i32 = dict(device="cuda", dtype=torch.int32)
    k, v = torch.zeros(64, nkv, page, dim, device="cuda", dtype=torch.bfloat16), torch.zeros(64, nkv, page, dim, device="cuda", dtype=torch.bfloat16)
    table = torch.arange(30, **i32).view(B, 10)
    ang = torch.rand(200, dim, device="cuda", generator=gen)
    cos, sin = ang.cos(), ang.sin()
    weights = torch.zeros(B, nkv, 160, device="cuda")
    prompts = [70, 9, 41]
    lens = torch.tensor(prompts, **i32)
    T = sum(prompts)
    qkv = torch.randn(T, 12 * dim, device="cuda", generator=gen).bfloat16()
    slots = torch.cat([torch.arange(n, **i32) for n in prompts])
    seqs = torch.cat([torch.full((n,), b, **i32) for b, n in enumerate(prompts)])
    int4_b200.paged_kv_append(qkv, cos, sin, slots, slots, table, k, v, seqs=seqs)
    positions = lens.clone()
    for step in range(40):
        qkv = torch.randn(B, 12 * dim, device="cuda", generator=gen).bfloat16()
        q = int4_b200.paged_kv_append(qkv, cos, sin, positions, lens, table, k, v)
        lens, positions = lens + 1, positions + 1
        ref, mag, wref, eps = _reference(q, k, v, table, lens)
        w0 = weights.double()
        out = int4_b200.paged_decode_attention(q, k, v, table, lens, weights=weights)
        assert ((out.double() - ref).abs() <= (_half(q.dtype) * 1.01 + 2 * eps) * (mag + ref.abs())).all()
        want = w0[..., :wref.shape[2]] + wref
        assert ((weights.double() - want).abs() <= wref * (2 * eps + 2 ** -20) + 2 ** -23 * want).all()
        if step % 15 == 14:  # cut to 48 slots, in the pages that the previous table does not use
            new = torch.arange(30, 60, **i32).view(B, 10) if table[0, 0] < 30 else torch.arange(30, **i32).view(B, 10)
            lens, kept, weights = int4_b200.paged_evict(weights, lens, table, k, v, new, 48, recent=8)
            table = new
            assert (lens <= 48).all()
