"""Paged steps as a server makes them: rows without a sequence, and a host that never waits for the GPU."""
from __future__ import annotations

import pytest
import torch

from test_decode_gpu import build_hf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda_device):
    from int4_b200.decode import LlamaTP

    return LlamaTP(build_hf(), w4=True, max_seq=128)


def _ids(n, seed):
    return torch.randint(0, 512, (1, n), generator=torch.Generator().manual_seed(seed)).cuda()


@torch.no_grad()
def test_tokens_of_rows_without_a_sequence_are_not_read(model):
    """Padding of any kind in the rows of sequences that are not live: the live rows' logits are the same bits."""
    caches = [model.paged_cache(32, max_seqs=4, page_size=8, max_len=96) for _ in range(2)]
    for c in caches:
        model.prefill_paged(_ids(11, 1), c, 1)
        model.prefill_paged(_ids(30, 2), c, 2)
    for step, pad in enumerate((-1, -100, 512, 2 ** 40)):
        tok = torch.tensor([[0], [7 + step], [400 - step], [0]], device="cuda")
        want = model.decode_paged(tok, caches[0])
        tok[0], tok[3] = pad, pad
        got = model.decode_paged(tok, caches[1])
        assert torch.isfinite(got).all() and torch.equal(got[1:3], want[1:3])
        assert tok[0, 0] == pad  # the caller's tensor is left as it is
