"""Refusals that need a device, and calls on tensors of which parts are missing or in use elsewhere."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_workspace_statuses(cuda_device):
    from int4_b200 import _lib

    L = _lib.lib()
    k = torch.zeros(40, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(2, 20, device="cuda", dtype=torch.int32)
    lens = torch.zeros(2, device="cuda", dtype=torch.int32)
    q = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.ones_like(q)
    ks = k.stride()
    c = _lib.PAGED_CACHE.pack(k.data_ptr(), k.data_ptr(), *ks[:3], *ks[:3], table.data_ptr(), 20, 40, 2, 16, 64, 2, 20, 1)
    need = L.i4b_paged_attention_workspace_size(2, 8, 2, 64, 320, 0)
    assert need > 0 and L.i4b_paged_attention_workspace_size(2, 8, 2, 64, 320, 1) > need
    assert L.i4b_paged_attention_workspace_size(2, 8, 2, 64, 256, 0) == 0  # whole items: nothing to keep
    assert L.i4b_paged_attention_workspace_size(2, 7, 2, 64, 320, 0) == 0  # not supported
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call(ws_ptr, size):
        return L.i4b_paged_decode_attention(c, q.data_ptr(), 512, 64, 8, lens.data_ptr(), 0.125, out.data_ptr(), None, 0, 0, ws_ptr, size, None)

    assert call(None, need) == 1 and call(ws.data_ptr(), need - 1) == 5 and (out == 1).all()
    assert call(ws.data_ptr(), need) == 0
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_operators_of_two_devices_are_refused(cuda_device):
    import int4_b200

    k = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(2, 2, dtype=torch.int32)
    lens = torch.zeros(2, device="cuda", dtype=torch.int32)
    q = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one device"):
        int4_b200.paged_decode_attention(q, k, k, table, lens)
    with pytest.raises(ValueError, match="one device"):
        int4_b200.token_logprobs(q, torch.zeros(2, 8, dtype=torch.int64))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_operators_on_a_device_that_is_not_the_current_one(cuda_device):
    import int4_b200

    z = torch.randn(3, 5000, device="cuda:1")
    t = torch.arange(3, device="cuda:1")
    lp, *_ = int4_b200.token_logprobs(z, t, top=2)
    torch.testing.assert_close(lp, torch.log_softmax(z, 1).gather(1, t[:, None])[:, 0], rtol=1e-5, atol=1e-5)


def test_attention_of_one_position_is_its_value(cuda_device):
    """One slot: every probability is exactly 1, every output exactly that slot's values, every weight the group's size."""
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(1)
    for dtype in (torch.bfloat16, torch.float16):
        for dim in (64, 128):
            k = torch.randn(8, 2, 8, dim, device="cuda", generator=gen).to(dtype)
            v = torch.randn(8, 2, 8, dim, device="cuda", generator=gen).to(dtype)
            table = torch.tensor([[3], [5], [0]], device="cuda", dtype=torch.int32)
            lens = torch.tensor([1, 1, 1], device="cuda", dtype=torch.int32)
            q = torch.randn(3, 6, dim, device="cuda", generator=gen).to(dtype)
            w = torch.zeros(3, 2, 8, device="cuda")
            out = int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w)
            want = v[table[:, 0].long(), :, 0].repeat_interleave(3, dim=1)
            assert torch.equal(out, want)
            assert (w[..., 0] == 3).all() and (w[..., 1:] == 0).all()


@pytest.mark.parametrize("cap_pages", [3, 40])  # whole items; split runs
def test_attention_tables_wider_than_the_sequences(cuda_device, cap_pages):
    """Entries behind a sequence's last page are never followed, whatever they hold; negative and huge lengths are clamped."""
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(2)
    k = torch.randn(16, 1, 16, 64, device="cuda", generator=gen).bfloat16()
    v = torch.randn(16, 1, 16, 64, device="cuda", generator=gen).bfloat16()
    q = torch.randn(3, 4, 64, device="cuda", generator=gen).bfloat16()
    table = torch.full((3, cap_pages), 2 ** 30, device="cuda", dtype=torch.int32)
    table[:, :3] = torch.arange(9, device="cuda", dtype=torch.int32).view(3, 3)
    lens = torch.tensor([40, -2 ** 31, 17], device="cuda", dtype=torch.int32)
    out = int4_b200.paged_decode_attention(q, k, v, table, lens)
    for b, n in ((0, 40), (2, 17)):
        kk, vv = k[table[b, :3].long(), 0].reshape(-1, 64)[:n].double(), v[table[b, :3].long(), 0].reshape(-1, 64)[:n].double()
        p = torch.softmax(q[b].double() @ kk.T / 8, -1)
        # the output's rounding, and what fp32 scores of at most 64 * |q||k| products leave
        assert ((out[b].double() - p @ vv).abs() <= 2 ** -8 * (p @ vv).abs() + 2 ** -14 * (p @ vv.abs())).all()
    assert (out[1] == 0).all()


def test_evict_of_rows_of_a_wider_tensor_and_two_calls_at_once(cuda_device):
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(3)
    big = torch.rand(2, 3, 2, 4100, device="cuda", generator=gen)
    w = big[0, :, :, 1:4097]  # rows that start off a 16-byte boundary
    k = torch.randn(256 * 3 + 3 * 70 * 2, 2, 16, 64, device="cuda", generator=gen).bfloat16()
    v = k.flip(0).contiguous()
    table = torch.arange(768, device="cuda", dtype=torch.int32).view(3, 256)
    lens = torch.tensor([4096, 1000, 4000], device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    results = []
    torch.cuda.synchronize()
    for i, stream in enumerate((torch.cuda.current_stream(), side)):
        new = (768 + 210 * i + torch.arange(210, device="cuda", dtype=torch.int32)).view(3, 70)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            results.append((int4_b200.paged_evict(w, lens, table, k, v, new, 1111, recent=77), new))
    torch.cuda.synchronize()
    for (n, kept, wo), new in results:
        assert n.tolist() == [1111, 1000, 1111]
        for b, L in enumerate((4096, 1000, 4000)):
            for h in range(2):
                m = min(L, 1111)
                if L > 1111:
                    best = torch.argsort(w[b, h, :L - 77], descending=True, stable=True)[:1111 - 77].sort().values
                    want = torch.cat([best, torch.arange(L - 77, L, device="cuda")])
                else:
                    want = torch.arange(L, device="cuda")
                assert torch.equal(kept[b, h, :m].long(), want) and (kept[b, h, m:] == -1).all()
                assert torch.equal(wo[b, h, :m], w[b, h, want]) and (wo[b, h, m:] == 0).all()
                at = torch.arange(m, device="cuda")
                assert torch.equal(k[new[b].long()[at // 16], h, at % 16], k[table[b].long()[want // 16], h, want % 16])
                assert torch.equal(v[new[b].long()[at // 16], h, at % 16], v[table[b].long()[want // 16], h, want % 16])


def test_evict_captured_and_replayed_with_other_lengths(cuda_device):
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(4)
    w = torch.rand(2, 2, 320, device="cuda", generator=gen)
    k = torch.randn(60, 2, 16, 64, device="cuda", generator=gen).bfloat16()
    v = torch.randn(60, 2, 16, 64, device="cuda", generator=gen).bfloat16()
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
    new = (40 + torch.arange(10, device="cuda", dtype=torch.int32)).view(2, 5)
    lens = torch.tensor([320, 100], device="cuda", dtype=torch.int32)
    int4_b200.paged_evict(w, lens, table, k, v, new, 70, recent=9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = int4_b200.paged_evict(w, lens, table, k, v, new, 70, recent=9)
    for a, b in ((320, 100), (71, 0), (5, 319)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        w.uniform_(generator=gen)
        g.replay()
        kept = k[new.long()].clone()
        want = int4_b200.paged_evict(w, lens, table, k, v, new, 70, recent=9)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(kept, k[new.long()])


def test_logprobs_on_two_streams_at_once(cuda_device):
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(5)
    z = (3 * torch.randn(5, 128256, device="cuda", generator=gen)).bfloat16()
    t = torch.arange(5, device="cuda")
    want = int4_b200.token_logprobs(z, t, top=7)
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got += [int4_b200.token_logprobs(z, t, top=7) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_scores_that_grow_and_shrink(cuda_device, dtype):
    """Scores that rise by hundreds along the sequence, fall, or are all alike; values near the type's range; a negative scale."""
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(6)
    n, dim, page = 700, 64, 16
    pages = -(-n // page)
    for kind in ("rising", "falling", "flat", "steps"):
        ramp = {"rising": torch.arange(n) * 0.5, "falling": -torch.arange(n) * 0.5, "flat": torch.zeros(n),
                "steps": (torch.arange(n) // 64 % 3) * 6.0}[kind].cuda()
        kk = torch.randn(n, dim, device="cuda", generator=gen)
        kk[:, 0] = ramp
        q = torch.randn(1, 4, dim, device="cuda", generator=gen)
        q[..., 0] = 4.0
        q = q.to(dtype)
        big = 1e36 if dtype == torch.bfloat16 else 6e4
        v0 = torch.rand(n, dim, device="cuda", generator=gen) * big
        k = torch.zeros(pages, 1, page, dim, device="cuda", dtype=dtype)
        v = torch.zeros_like(k)
        k.view(-1, dim)[:n], v.view(-1, dim)[:n] = kk.to(dtype), v0.to(dtype)
        table = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
        lens = torch.tensor([n], device="cuda", dtype=torch.int32)
        for scale in (0.125, -0.125, 1.0):
            w = torch.zeros(1, 1, pages * page, device="cuda")
            out = int4_b200.paged_decode_attention(q, k, v, table, lens, scale=scale, weights=w)
            kd, vd = k.view(-1, dim)[:n].double(), v.view(-1, dim)[:n].double()
            s = q[0].double() @ kd.T * scale
            p = torch.softmax(s, -1)
            # fp32 scores: 64 products and sums, the scale and the subtraction, at the size of the largest
            eps = (dim + 8) * 2 ** -24 * float((q[0].double().abs() @ kd.abs().T).max()) * abs(scale) * 2 + 2 ** -20
            half = torch.finfo(dtype).eps / 2
            ref = p @ vd
            # fp16 holds a probability as two numbers down to 2^-24 of the range's top: n of them, each off by 2^-25 at most
            small = n * 2 ** -25 * float(vd.max()) * (1 if dtype == torch.float16 else 0)
            assert torch.isfinite(out).all()
            assert ((out[0].double() - ref).abs() <= half * ref + 2 * eps * ref + small).all(), (kind, scale)
            assert ((w[0, 0, :n].double() - p.sum(0)).abs() <= p.sum(0) * (2 * eps + 2 ** -20) + 2 ** -60).all(), (kind, scale)


def test_attention_output_may_take_the_queries_place(cuda_device):
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(7)
    for cap in (12, 300):
        k = torch.randn(cap * 2, 2, 16, 64, device="cuda", generator=gen).bfloat16()
        v = torch.randn(cap * 2, 2, 16, 64, device="cuda", generator=gen).bfloat16()
        table = torch.arange(cap * 2, device="cuda", dtype=torch.int32).view(2, cap)
        lens = torch.tensor([cap * 16, cap * 16 - 37], device="cuda", dtype=torch.int32)
        q = torch.randn(2, 8, 64, device="cuda", generator=gen).bfloat16()
        want = int4_b200.paged_decode_attention(q, k, v, table, lens)
        assert torch.equal(int4_b200.paged_decode_attention(q, k, v, table, lens, out=q), want)


@pytest.mark.parametrize("cap_pages", [3, 80])  # whole items; split runs
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 30.0), (torch.bfloat16, 3.3e3), (torch.bfloat16, 1e9), (torch.float16, 1.7e3),
                                        (torch.float16, 6e4)])
def test_attention_of_large_scores(cuda_device, dtype, size, cap_pages):
    """One slot's score, or two equal ones, far above all others: probabilities of 1, or of 1/2 each, at any size of the
    scores; the others' are 0 (the smallest distance is 64 * 30 * 30 * 0.125 / 2 = 3600).  All of this is exact."""
    import int4_b200

    B, nkv, G, dim, ps = 3, 2, 4, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(5)
    pages = B * cap_pages
    k = torch.full((pages, nkv, ps, dim), -size, device="cuda").to(dtype)
    v = torch.randn(pages, nkv, ps, dim, device="cuda", generator=gen).to(dtype)
    table = torch.randperm(pages, device="cuda", generator=gen).int().view(B, cap_pages)
    lens = torch.tensor([cap_pages * ps, cap_pages * ps - 5, 37], device="cuda", dtype=torch.int32)
    q = torch.full((B, nkv * G, dim), size, device="cuda").to(dtype)
    w = torch.zeros(B, nkv, cap_pages * ps, device="cuda")
    want_w, want = w.clone(), torch.empty(B, nkv, dim, device="cuda")
    for b in range(B):
        for h in range(nkv):
            at = [7, 36] if h else [int(lens[b]) - 3]
            for j in at:
                k[table[b, j // ps].long(), h, j % ps] = torch.tensor(size / 2).to(dtype)
                want_w[b, h, j] = G / len(at)
            want[b, h] = sum(v[table[b, j // ps].long(), h, j % ps].float() for j in at) / len(at)
    out = int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w)
    assert torch.equal(out, want.to(dtype).repeat_interleave(G, dim=1))
    assert torch.equal(w, want_w)
