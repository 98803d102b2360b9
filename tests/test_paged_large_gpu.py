"""The attention's forms for large batches: runs taken from a counter, a warp per head in the join, and both values of a
probability.

Tolerances.  ``eps`` bounds a probability's relative error in fp32: dim + 8 roundings of a score, twice (its own and the
maximum's), and 2^-20 for the exponential and the joins' factors.  A run sums at most 64 tiles, 8 additions each, relative to
sum p |v|: 512 half steps.  A probability is the sum of two values of the cache's type: within half^2 of itself (fp16: or
2^-51).  The output is rounded once: half a step of it.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2 ** -24


def _filled(lens, nq, nkv, dim, page, dtype, seed, width=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = width or max(need)
    pages = sum(need) + 1
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.empty(pages, nkv, page, dim, device="cuda", dtype=dtype).normal_(generator=gen) for _ in "kv")
    q = torch.empty(len(lens), nq, dim, device="cuda", dtype=dtype).normal_(std=1.5, generator=gen)
    return q, k, v, table, torch.tensor(lens, device="cuda", dtype=torch.int32)


def _check(out, w, q, k, v, table, lens):
    B, nq, dim = q.shape
    nkv, page = k.shape[1:3]
    G, half, scale = nq // nkv, torch.finfo(q.dtype).eps / 2, dim ** -0.5
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            assert (out[b] == 0).all() and (w is None or (w[b] == 0).all())
            continue
        rows = table[b, :-(-n // page)].long()
        kk, vv = (x[rows].transpose(0, 1).reshape(nkv, -1, dim)[:, :n].double() for x in (k, v))
        qq = q[b].view(nkv, G, dim).double()
        p = torch.softmax(qq @ kk.transpose(1, 2) * scale, -1)
        worst = float((qq.abs() @ kk.abs().transpose(1, 2)).max()) * scale
        eps = (dim + 8) * STEP * worst * 2 + 2 ** -20
        ref, mag = p @ vv, p @ vv.abs()
        lost = n * 2.0 ** -51 * float(vv.abs().max())
        tol = half * ref.abs() + 1.01 * (2 * eps + 512 * STEP + half * half) * mag + lost
        err = (out[b].view(nkv, G, dim).double() - ref).abs()
        assert (err <= tol).all(), (b, n, float((err / tol).max()))
        if w is not None:
            want = p.sum(1)
            assert ((w[b, :, :n].double() - want).abs() <= want * (2 * eps + (512 + G) * STEP)).all(), (b, n)
            assert (w[b, :, n:] == 0).all()


def _run(q, k, v, table, lens, with_weights):
    import int4_b200

    w = torch.zeros(q.shape[0], k.shape[1], table.shape[1] * k.shape[2], device="cuda") if with_weights else None
    return int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w), w


# A short run has `last` tiles, 2 or as many as 4 KB of outputs ask for; runs are shared from 8 `last` tiles per warp on
# (1480 warps on 148 SMs): 23680 tiles of 32 slots for up to 8 heads of 64, 94720 of 16 for 16 heads of 128.
LONG = [20000, 0, 16384, 1, 16001, 9000, 20003, 17000]
SHARED = [(LONG, 32, 8, 64, 64), ([35000] * 3 + [0, 31, 33000, 34567, 24999], 128, 8, 64, 128),
          ([32000, 31999, 33234, 30001, 0, 31888, 34000, 17], 128, 8, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,nq,nkv,dim,page", SHARED)
@pytest.mark.parametrize("with_weights", [False, True])
def test_runs_from_the_counter(cuda_device, dtype, lens, nq, nkv, dim, page, with_weights):
    args = _filled(lens, nq, nkv, dim, page, dtype, seed=nq + dim)
    tile = 2048 // dim
    last = max(2, min(16, nq // nkv) * dim * 4 * 8 // 8192)
    warps = 10 * torch.cuda.get_device_properties(0).multi_processor_count
    assert sum(-(-n // tile) for n in lens) * nkv * -(-(nq // nkv) // 16) >= warps * 8 * last  # the sizes do what the test is for
    out, w = _run(*args, with_weights)
    _check(out, w, *args)
    for _ in range(5):  # whichever warp takes which run
        again, w2 = _run(*args, with_weights)
        assert torch.equal(out, again) and (w is None or torch.equal(w, w2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,nq,nkv,dim,page,longest", [
    (20, 32, 8, 64, 16, 600),      # at least 512 heads, up to 128 tiles: a warp per head
    (16, 32, 4, 128, 16, 300),
    (20, 32, 2, 64, 64, 5000),     # 512 heads, more tiles: 128 threads per head
    (70, 32, 2, 64, 64, 4400),     # 2048 heads: a warp per head
    (65, 32, 2, 128, 32, 2300)])
@pytest.mark.parametrize("with_weights", [False, True])
def test_joins_of_many_heads(cuda_device, dtype, B, nq, nkv, dim, page, longest, with_weights):
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(1, longest, (B,), generator=gen).tolist()
    lens[0], lens[3], lens[B // 2], lens[-1] = longest, 0, 1, 0
    args = _filled(lens, nq, nkv, dim, page, dtype, seed=B + dim)
    assert args[3].shape[1] * page > 8 * (2048 // dim)  # more than whole items
    out, w = _run(*args, with_weights)
    _check(out, w, *args)
    again, w2 = _run(*args, with_weights)
    assert torch.equal(out, again) and (w is None or torch.equal(w, w2))


@pytest.mark.parametrize("with_weights", [False, True])
def test_one_graph_with_and_without_shared_runs(cuda_device, with_weights):
    """Lengths on either side of the threshold, replayed in one graph on two streams' data at once."""
    import int4_b200

    states = []
    for i in range(2):
        q, k, v, table, lens = _filled(LONG, 32, 8, 64, 64, torch.bfloat16, seed=40 + i)
        w = torch.zeros(len(LONG), 8, table.shape[1] * 64, device="cuda") if with_weights else None
        out = torch.empty_like(q)
        int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            int4_b200.paged_decode_attention(q, k, v, table, lens, weights=w, out=out)
        states.append((q, k, v, table, lens, w, out, g, torch.cuda.Stream()))
    for now in (LONG, [n // 2 for n in LONG], [0] * 8, [min(n, 40) for n in LONG], LONG):
        for q, k, v, table, lens, w, out, g, s in states:
            lens.copy_(torch.tensor(now, dtype=torch.int32))
            if w is not None:
                w.zero_()
        torch.cuda.synchronize()
        for n in range(6):
            for q, k, v, table, lens, w, out, g, s in states:
                with torch.cuda.stream(s):
                    if w is not None:
                        w.zero_()
                    g.replay()
        torch.cuda.synchronize()
        for q, k, v, table, lens, w, out, g, s in states:
            want, w2 = _run(q, k, v, table, lens, with_weights)
            assert torch.equal(out, want) and (w is None or torch.equal(w, w2))
            _check(out, w, q, k, v, table, lens)


def _pairs(dtype, B, nkv, page, width, gen, device):
    """Scores and values of rows of two slots: probabilities 1 and p relative to the larger, values round(p) and -1."""
    s = torch.empty(B * width, nkv, page, device=device).uniform_(0.5, 1.5, generator=gen).to(dtype)
    s[:, :, 1::2] = (s[:, :, 0::2].float() - torch.empty_like(s[:, :, 1::2], dtype=torch.float32).uniform_(0.05, 0.6, generator=gen)).to(dtype)
    v = torch.full_like(s, -1)
    v[:, :, 0::2] = (s[:, :, 1::2].double() - s[:, :, 0::2].double()).exp().to(dtype)
    return s, v


def _pair_reference(s, v, dtype):
    """Outputs of rows of two slots in 64 bits, and the bound of an output's error.

    Scores are exact and below 1.5: a probability is off by the roundings of three numbers below 2.2 (units of log 2) and by
    2^-22 of the exponential, 2^-20 in all, and so is the sum; 8 half steps for the four sums and products."""
    half = torch.finfo(dtype).eps / 2
    p = torch.softmax(s.double(), -1)
    ref = (p * v.double()).sum(-1)
    return ref, half * ref.abs() + half * half + 2 * 2 ** -20 + 8 * STEP + torch.finfo(dtype).smallest_normal * half


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,G,width", [(64, 4, 4), (64, 16, 40), (128, 8, 4), (128, 16, 40)])
def test_probabilities_have_two_values(cuda_device, dtype, dim, G, width):
    """Values that leave of an output what rounding leaves of a probability: one rounded once to the cache's type would
    give 0 (shown for the oracle at the end)."""
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(dim + G)
    page, B, nkv = 16, 96, 2
    s, sign = _pairs(dtype, B, nkv, page, width, gen, "cuda")
    k = torch.zeros(B * width, nkv, page, dim, device="cuda", dtype=dtype)
    k[..., 3] = s
    v = sign[..., None].expand(k.shape).contiguous()
    table = torch.randperm(B * width, device="cuda", generator=gen).to(torch.int32).view(B, width)
    lens = torch.full((B,), 2, device="cuda", dtype=torch.int32)
    q = torch.zeros(B, nkv * G, dim, device="cuda", dtype=dtype)
    q[..., 3] = 1
    out = int4_b200.paged_decode_attention(q, k, v, table, lens, scale=1.0)
    ss, vv = (x[table[:, 0].long(), :, :2] for x in (s, sign))
    ref, tol = _pair_reference(ss, vv, dtype)
    err = (out.view(B, nkv, G, dim).double() - ref[:, :, None, None]).abs()
    assert (err <= tol[:, :, None, None]).all(), (float(err.max()), float(tol.max()))
    p = (ss.double() - ss.double().amax(-1, keepdim=True)).exp()
    once = (p.to(dtype).double() * vv.double()).sum(-1) / p.sum(-1)
    assert ((once - ref).abs() > 4 * tol).float().mean() > 0.25
