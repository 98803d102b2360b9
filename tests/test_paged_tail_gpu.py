"""Attention rows whose small probabilities carry the output: one slot far above the others, with a value of 0.

Every key has one number that is not 0 and the scale is 1, so a score is exact.  A probability's relative error is then
that of its exponential: the conversion to units of log 2, the product's and the difference's roundings of numbers up to
``gap * log2(e)``, at most 6 * gap half steps of fp32 in units of the probability, and 2^-22 of the exponential itself.
The sums (a run's tiles, then the runs) add at most 512 half steps, the joins' factors 2^-20.  A probability enters the
product with the values as two numbers of the cache's type, within half^2 of itself, for fp16 no closer than 2^-51.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2 ** -24


def _rows(dtype, dim, n, width, page, gap, nkv, G, seed, B=2):
    """B sequences of n, n - 3, n, ... slots: scores of about 0, one of ``gap``; values of about 0.5, there 0."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = B * width
    k = torch.zeros(pages, nkv, page, dim, device="cuda", dtype=dtype)
    v = torch.rand(pages, nkv, page, dim, device="cuda", generator=gen).to(dtype)
    k[..., 5] = (0.3 * torch.randn(pages, nkv, page, device="cuda", generator=gen)).to(dtype)
    table = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).view(B, width)
    lens = torch.tensor([n - 3 * (b % 2) for b in range(B)], device="cuda", dtype=torch.int32)
    for b in range(B):
        at = 11 if b % 2 == 0 else n - 4
        k[table[b, at // page].long(), :, at % page, 5] = gap
        v[table[b, at // page].long(), :, at % page] = 0.0
    q = torch.zeros(B, nkv * G, dim, device="cuda", dtype=dtype)
    q[..., 5] = 1.0
    return q, k, v, table, lens


def _check(q, k, v, table, lens, gap, with_weights):
    import int4_b200

    B, nq, dim = q.shape
    nkv, page = k.shape[1:3]
    w = torch.zeros(B, nkv, table.shape[1] * page, device="cuda") if with_weights else None
    out = int4_b200.paged_decode_attention(q, k, v, table, lens, scale=1.0, weights=w)
    half = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * half  # half the distance of two subnormal numbers
    eps = 6 * gap * STEP + 2 ** -22 + 512 * STEP + 2 ** -20
    for b in range(B):
        n = int(lens[b])
        rows = table[b].long()
        kk = k[rows].transpose(0, 1).reshape(nkv, -1, dim)[:, :n]
        vv = v[rows].transpose(0, 1).reshape(nkv, -1, dim)[:, :n].double()
        for h in range(nkv):
            p = torch.softmax(kk[h, :, 5].double(), 0)
            ref = p @ vv[h]
            lost = n * 2.0 ** -51 * float(vv[h].max()) if q.dtype == torch.float16 else 0.0
            tol = half * ref + 1.01 * (2 * eps + half * half) * ref + lost + tiny
            heads = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            err = (out[b, heads].double() - ref).abs()
            assert (err <= tol).all(), (b, h, float((err / ref.clamp(min=1e-300)).max()), float((tol / ref.clamp(min=1e-300)).min()))
            if with_weights:
                want = p * (nq // nkv)
                assert ((w[b, h, :n].double() - want).abs() <= want * (2 * eps + 2 ** -20)).all()
                assert (w[b, h, n:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,G", [(64, 4), (64, 12), (128, 8), (128, 16)])
@pytest.mark.parametrize("gap", [5.0, 10.0, 14.0, 18.0])
@pytest.mark.parametrize("with_weights", [False, True])
def test_tail_of_a_short_row(cuda_device, dtype, dim, G, gap, with_weights):
    _check(*_rows(dtype, dim, 125, 8, 16, gap, 2, G, int(gap) + G), gap, with_weights)  # whole items


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,G", [(64, 4), (128, 8), (64, 16)])
@pytest.mark.parametrize("n,gap", [(1000, 14.0), (1000, 18.0), (131073, 12.0), (131073, 18.0), (131073, 26.0)])
@pytest.mark.parametrize("with_weights", [False, True])
def test_tail_of_a_long_row(cuda_device, dtype, dim, G, n, gap, with_weights):
    _check(*_rows(dtype, dim, n, -(-n // 64), 64, gap, 1, G, int(gap) + G), gap, with_weights)  # split and joined


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,G", [(64, 4), (64, 16), (128, 8)])
@pytest.mark.parametrize("gap", [10.0, 14.0, 18.0, 21.0, 28.0])
@pytest.mark.parametrize("with_weights", [False, True])
def test_tail_within_long_runs(cuda_device, dtype, dim, G, gap, with_weights):
    """So many sequences that one warp goes through most of a row: nothing but the running sums holds its tail."""
    _check(*_rows(dtype, dim, 3001, 47, 64, gap, 8, G, int(gap) + G, B=40), gap, with_weights)
