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


@torch.no_grad()
def test_the_host_does_not_wait_for_the_gpu(model):
    """Prompts, steps that take new pages, an eviction and a freed sequence, under torch's check for synchronising calls."""

    def run(cache):
        model.prefill_paged(prompts[0], cache, 0)
        model.prefill_paged(prompts[1][:, :13], cache, 2)
        model.prefill_paged(prompts[1][:, 13:], cache, 2)
        out = [model.decode_paged(tok, cache) for _ in range(20)]
        cache.evict(24, recent=4)
        out.append(model.decode_paged(tok, cache))
        cache.free(0)
        model.prefill_paged(prompts[0], cache, 1)
        out.append(model.decode_paged(tok, cache))
        return torch.stack([x[2] for x in out])

    prompts, tok = [_ids(23, 3), _ids(30, 4)], torch.ones(3, 1, dtype=torch.long, device="cuda")
    caches = [model.paged_cache(40, max_seqs=3, page_size=8, max_len=96, track_weights=True) for _ in range(2)]
    want = run(caches[0])  # what is set up by the first calls may wait
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = run(caches[1])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(got, want)
    a, b = caches
    assert a.pages == b.pages and a.lengths == b.lengths == b.lens.tolist() and a.seen == b.seen == b.positions.tolist()
    assert b.live.tolist() == [0, 1, 1] and torch.equal(a.table, b.table) and torch.equal(a.weights, b.weights)
    for seq in range(3):
        n = len(b.pages[seq])
        assert b.table[seq].tolist() == b.pages[seq] + [-1] * (b.table.shape[1] - n)
