"""token_logprobs against torch.log_softmax in 64 bits.

Tolerance of a log probability: the sum of n exponentials in fp32 (a thread adds n / 512 of them at most, then a tree)
is off by (n / 512 + 64) half steps relatively, each exponential by its argument's rounding (its size times half a
step) and a few units of the exponential; then a few roundings of numbers of the size of the logits.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2 ** -24


def _check(logits, targets, top):
    import int4_b200

    lp, entropy, top_lp, top_ids = int4_b200.token_logprobs(logits, targets, top=top)
    assert lp.dtype == entropy.dtype == torch.float32 and lp.shape == entropy.shape == targets.shape
    z = logits.double().reshape(-1, logits.shape[-1])
    t, n = targets.reshape(-1), logits.shape[-1]
    none = (z == -math.inf).all(1)
    ref = torch.where(none[:, None], -math.inf, torch.log_softmax(z, 1))
    p = ref.exp()
    want = torch.where(t < 0, 0.0, ref.gather(1, t.clamp(0, n - 1)[:, None])[:, 0])
    finite = torch.where(z.isfinite(), z.abs(), 0.0)
    size = finite.max(1).values + math.log(n) + 1
    # exponentials of far smaller logits weigh nothing: what an argument's rounding costs is sum p |d| half steps
    h = -torch.where(p > 0, p * ref, 0.0).sum(1)
    rel = (n / 512 + 96) * STEP + 4 * STEP * (h + 4) + 2 ** -21
    tol = rel + 4 * STEP * size
    same = (lp.reshape(-1).double() == want) | ((lp.reshape(-1).double() - want).abs() <= tol + 2 * STEP * want.abs())
    assert same.all(), (lp.reshape(-1)[~same], want[~same])
    assert ((entropy.reshape(-1).double() - h).abs() <= 2 * tol * (1 + h)).all()
    if top:
        order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :top]
        assert top_ids.dtype == torch.int64 and top_ids.shape == (*targets.shape, top)
        assert torch.equal(top_ids.reshape(-1, top), order)
        w = ref.gather(1, order)
        got = top_lp.reshape(-1, top).double()
        assert ((got == w) | ((got - w).abs() <= tol[:, None] + 2 * STEP * w.abs())).all()
    else:
        assert top_lp is None and top_ids is None


def _logits(rows, n, dtype, seed=0, std=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + n)
    z = (std * torch.randn(rows, n, device="cuda", generator=gen)).to(dtype)
    return z, torch.randint(0, n, (rows,), device="cuda", generator=gen)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (2, 7, 7), (3, 33, 32), (5, 1000, 5), (1, 128256, 20), (17, 50257, 1), (300, 4099, 3),
                                        (40, 32000, 0), (1, 200001, 32), (9, 513, 32)])
def test_matches_log_softmax(cuda_device, dtype, rows, n, top):
    _check(*_logits(rows, n, dtype), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 400])
def test_masked_rows(cuda_device, dtype, rows):
    z, t = _logits(rows, 5003, dtype, 1)
    z[0, 3:] = -math.inf  # fewer tokens left than alternatives
    t[0] = 2
    z[1] = -math.inf  # nothing left
    if rows > 2:
        z[2, 7:] = torch.finfo(dtype).min  # masked by the type's lowest value
        z[3] = torch.finfo(dtype).min
        z[4, :] = 1.5  # all alike
        z[5, 100:] = -math.inf
        z[6] = torch.arange(5003, device="cuda").to(dtype) / 100  # ordered, with ties in 16 bits
        z[7] = -z[6]
        z[8, ::512] = 90.0
        z[9, :40] = 50.0
        t[10], t[11] = -1, -100
        t[12] = 0
        z[12, 0] = -math.inf  # a token that the mask rules out
    _check(z, t, 9)
    _check(z, t, 0)


def test_ties_go_to_the_lowest_index(cuda_device):
    for n in (100, 5000, 128256):
        z = torch.zeros(3, n, device="cuda")
        z[0, n // 2:] = 1.0
        z[1, [5, n - 1, n // 3]] = 2.0
        z[2] = -0.0
        z[2, n // 2] = 0.0
        _check(z, torch.zeros(3, dtype=torch.int64, device="cuda"), 16)


def test_nan_and_positive_infinity(cuda_device):
    import int4_b200

    z, t = _logits(4, 3000, torch.float32, 2)
    want = int4_b200.token_logprobs(z, t, top=4)
    z[1, 77] = math.nan
    z[2, 78] = math.inf
    t[3] = 3000
    lp, entropy, top_lp, top_ids = int4_b200.token_logprobs(z, t, top=4)
    assert torch.isnan(lp[1:]).all() and torch.isnan(entropy[1:3]).all() and torch.isnan(top_lp[1:3]).all()
    assert lp[0] == want[0][0] and torch.equal(top_ids[1], want[3][1]) and top_ids[2, 0] == 78
    z[:] = math.nan
    _, _, top_lp, top_ids = int4_b200.token_logprobs(z, t, top=4)
    assert torch.isnan(top_lp).all() and ((top_ids >= 0) & (top_ids < 3000)).all()


def test_shapes_and_strides(cuda_device):
    z, t = _logits(12, 1003, torch.bfloat16, 3)
    wide = torch.zeros(12, 1011, device="cuda", dtype=torch.bfloat16)
    wide[:, 5:1008] = z
    _check(wide[:, 5:1008], t, 4)  # rows that start anywhere
    _check(z.view(3, 4, 1003), t.view(3, 4), 4)
    _check(z.t().contiguous().t(), t, 4)
    _check(z[:1].expand(5, 1003), t[:5], 4)
    _check(wide[::3, 5:1008], t[::3], 2)
    import int4_b200

    lp, entropy, top_lp, top_ids = int4_b200.token_logprobs(z[:0], t[:0], top=3)
    assert lp.shape == (0,) and top_ids.shape == (0, 3)
    lp, *_ = int4_b200.token_logprobs(z[0], t[0])
    assert lp.shape == ()


def test_captured_and_replayed(cuda_device):
    import int4_b200

    z, t = _logits(4, 128256, torch.bfloat16, 4)
    int4_b200.token_logprobs(z, t, top=5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = int4_b200.token_logprobs(z, t, top=5)
    for seed in (5, 6):
        z2, t2 = _logits(4, 128256, torch.bfloat16, seed)
        z.copy_(z2), t.copy_(t2)
        g.replay()
        want = int4_b200.token_logprobs(z2, t2, top=5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("m", [1.0e3, 1.2345e5, 1.0e6, 12345678.0, 2.0 ** 40, 3.3e9, 1.1e20, 2.5e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_logits(cuda_device, dtype, m, rows):
    """k tokens share the largest logit, +m or -m, the others are far below: log probabilities -log k, entropy log k.

    Each of the k terms and the factor that puts a row's maximum right is an exponential of an argument up to 1 (off by
    2^-22 relatively); k <= 24 terms add at most 24 half steps, the products, quotients and the logarithm a few more:
    2^-21 + 40 * 2^-24 < 2^-18 with log 24 < 4."""
    import int4_b200

    n, k = 6001, [1, 2, 7, 24]
    gen = torch.Generator().manual_seed(int(math.log2(m)))
    z = torch.empty(rows, n, dtype=torch.float32)
    picked = []
    for r in range(rows):
        sign = 1.0 if r % 2 == 0 else -1.0
        z[r] = {0: -math.inf, 1: torch.finfo(dtype).min, 2: sign * m - 0.2 * m}[r // 2 % 3]
        at = torch.randperm(n, generator=gen)[: k[r % 4]].sort().values
        z[r, at] = sign * m
        picked.append(at)
    t = torch.tensor([int(at[-1]) for at in picked], device="cuda")
    lp, entropy, top_lp, top_ids = int4_b200.token_logprobs(z.to(dtype).cuda(), t, top=1)
    want = torch.tensor([math.log(len(at)) for at in picked], dtype=torch.float64)
    assert ((lp.cpu().double() + want).abs() <= 2.0 ** -18).all(), lp.cpu().double() + want
    assert ((top_lp[:, 0].cpu().double() + want).abs() <= 2.0 ** -18).all()
    assert ((entropy.cpu().double() - want).abs() <= 2.0 ** -18).all(), entropy.cpu().double() - want
    assert top_ids[:, 0].cpu().tolist() == [int(at[0]) for at in picked]
