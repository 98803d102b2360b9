"""token_logprobs where a row's largest logits are more than its lists hold."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 300])
@pytest.mark.parametrize("n", [102400, 102403, 8192])
def test_more_candidates_than_the_lists_hold(cuda_device, dtype, rows, n):
    """Every 32nd 16-byte chunk holds small logits alone, all others large ones: the 32nd largest of the 32 group maxima is
    small, and thousands of logits lie above it.  Few distinct values too, so that ties have to go to the lower index."""
    import int4_b200

    gen = torch.Generator(device="cuda").manual_seed(n + rows)
    vec = 16 // torch.finfo(dtype).bits * 8
    pitch = -(-n // 8) * 8
    z = torch.empty(rows, pitch, device="cuda").uniform_(5.0, 9.0, generator=gen).to(dtype)
    z[rows // 2] = torch.randint(2, 6, (pitch,), device="cuda", generator=gen).to(dtype)
    z.view(rows, -1)[:, torch.arange(pitch, device="cuda") // vec % 32 == 0] = -3.0
    z = z[:, :n]
    t = torch.randint(0, n, (rows,), device="cuda", generator=gen)
    lp, entropy, top_lp, top_ids = int4_b200.token_logprobs(z, t, top=32)
    ref = torch.log_softmax(z.double(), 1)
    order = torch.argsort(z.double(), dim=1, descending=True, stable=True)[:, :32]
    assert torch.equal(top_ids, order)
    # sums of n exponentials below 1 in fp32, n / 512 by each thread at most, then a tree; logits below 16
    tol = (n / 256 + 96) * 2 ** -24 + 2 ** -18
    assert ((top_lp.double() - ref.gather(1, order)).abs() <= tol).all()
    assert ((lp.double() - ref.gather(1, t[:, None])[:, 0]).abs() <= tol).all()
    assert ((entropy.double() + (ref.exp() * ref).sum(1)).abs() <= 16 * tol).all()
