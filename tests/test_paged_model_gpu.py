"""LlamaTP over a paged cache: the same model as over its static cache, for sequences of different lengths.

The paged step differs from the static one in two roundings (it rotates in fp32 and rounds once; its attention keeps
the probabilities exact), so the logits are held to the bound that the static step is held to against transformers,
2e-2 max-abs (``tests/test_decode_gpu.py``).
"""
from __future__ import annotations

import pytest
import torch

from test_decode_gpu import LOGIT_TOL, build_hf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hf(cuda_device):
    return build_hf()


def _ids(n, seed):
    return torch.randint(0, 512, (1, n), generator=torch.Generator().manual_seed(seed)).cuda()


@torch.no_grad()
@pytest.mark.parametrize("w4", [True, False])
@pytest.mark.parametrize("page", [8, 64])
def test_ragged_decode_matches_each_sequence_alone(hf, w4, page):
    from int4_b200.decode import LlamaTP

    m = LlamaTP(hf, w4=w4, max_seq=128)
    prompts = [_ids(n, n) for n in (40, 1, 17)]
    cache = m.paged_cache(64, max_seqs=4, page_size=page, max_len=128)
    rows = [0, 2, 3]  # row 1 stays empty
    last = {}
    for row, p in zip(rows, prompts):
        if p.shape[1] > 20:  # in two parts
            m.prefill_paged(p[:, :13], cache, row)
            last[row] = m.prefill_paged(p[:, 13:], cache, row)
        else:
            last[row] = m.prefill_paged(p, cache, row)
    steps = [torch.randint(0, 512, (4, 1), generator=torch.Generator().manual_seed(99 + s)).cuda() for s in range(10)]
    got = [m.decode_paged(t, cache) for t in steps]
    assert cache.lengths == [50, 0, 11, 27] and cache.lens.tolist() == cache.lengths == cache.positions.tolist()
    for row, p in zip(rows, prompts):
        ref = m.prefill(p)
        assert (last[row].float() - ref.float()).abs().max().item() <= LOGIT_TOL
        for s, t in enumerate(steps):
            ref = m.decode_step(t[row:row + 1], torch.tensor([p.shape[1] + s], device="cuda"))
            err = (got[s][row].float() - ref[0].float()).abs().max().item()
            assert err <= LOGIT_TOL, (row, s, err)


@torch.no_grad()
def test_paged_decode_replays_from_a_cuda_graph(hf):
    from int4_b200.decode import LlamaTP

    m = LlamaTP(hf, w4=True, max_seq=128)
    caches = [m.paged_cache(32, max_seqs=2, page_size=8, max_len=96, track_weights=True) for _ in range(2)]
    for c in caches:
        m.prefill_paged(_ids(11, 1), c, 0)
        m.prefill_paged(_ids(30, 2), c, 1)
    tok = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    eager = []
    for s in range(12):
        tok.fill_(s)
        eager.append(m.decode_paged(tok, caches[0]).clone())
    c = caches[1]
    state = [t.clone() for t in (c.lens, c.positions, c.weights)]
    c.reserve_step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.decode_paged(tok, c, reserve=False)  # warm-up: its slot is written again by the first replay
    torch.cuda.synchronize()
    for t, x in zip((c.lens, c.positions, c.weights), state):
        t.copy_(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = m.decode_paged(tok, c, reserve=False)
    for t, x in zip((c.lens, c.positions, c.weights), state):
        t.copy_(x)
    for s in range(12):
        if s:
            c.reserve_step()
        tok.fill_(s)
        g.replay()
        assert torch.equal(out, eager[s]), s
    assert c.lens.tolist() == caches[0].lens.tolist() == [23, 42]
    assert torch.equal(c.weights, caches[0].weights)


@torch.no_grad()
def test_bounded_decode_evicts_and_goes_on(hf):
    """Sequences cut at a budget: pages come back, lengths stay bounded, positions run on; the weights say what is kept."""
    from int4_b200.decode import LlamaTP

    m = LlamaTP(hf, w4=True, max_seq=256)
    cache = m.paged_cache(40, max_seqs=3, page_size=8, max_len=120, track_weights=True)
    m.prefill_paged(_ids(60, 5), cache, 0)
    m.prefill_paged(_ids(9, 6), cache, 2)
    tok = torch.ones(3, 1, dtype=torch.long, device="cuda")
    for step in range(100):
        out = m.decode_paged(tok, cache)
        assert torch.isfinite(out[[0, 2]]).all()
        if max(cache.lengths) > 64:
            before = {s: cache.weights[:, s].clone() for s in (0, 2)}
            old = list(cache.lengths)
            cut = cache.evict(48, recent=16)
            assert cut == [s for s in (0, 2) if old[s] > 48] and all(cache.lengths[s] == 48 for s in cut)
            for s in cut:
                now = cache.weights[:, s]
                assert (now[..., 48:] == 0).all()
                assert torch.equal(now[..., 32:48], before[s][..., old[s] - 16:old[s]])  # the recent ones
                heavy = before[s][..., :old[s] - 16].topk(32, dim=-1).values.sum(-1)
                torch.testing.assert_close(now[..., :32].sum(-1), heavy, rtol=32 * 2 ** -23, atol=0)
    assert cache.positions.tolist() == [160, 0, 109] and cache.lens.tolist() == cache.lengths
    used = sum(len(p) for p in cache.pages)
    assert used + len(cache.free_pages) == 40 and len(set(cache.free_pages) | {p for q in cache.pages for p in q}) == 40
    # every token's probabilities add up to one per query head: what a slot has received is never lost but by eviction
    cache.free(0)
    cache.free(2)
    assert sorted(cache.free_pages) == list(range(40)) and (cache.table == -1).all() and (cache.weights == 0).all()


@torch.no_grad()
def test_cache_refuses_what_does_not_fit(hf):
    from int4_b200._lib import Int4B200Error
    from int4_b200.decode import LlamaTP

    m = LlamaTP(hf, w4=True, max_seq=64)
    cache = m.paged_cache(4, max_seqs=2, page_size=8, max_len=24)
    with pytest.raises(Int4B200Error, match="slots"):
        m.prefill_paged(_ids(25, 1), cache, 0)
    m.prefill_paged(_ids(24, 1), cache, 0)
    with pytest.raises(Int4B200Error, match="pages"):
        m.prefill_paged(_ids(9, 1), cache, 1)
    assert cache.lengths == [24, 0] and len(cache.free_pages) == 1
    with pytest.raises(Int4B200Error, match="slots"):
        m.decode_paged(torch.zeros(2, 1, dtype=torch.long, device="cuda"), cache)
    with pytest.raises(ValueError, match="track_weights"):
        cache.evict(8)
    long = m.paged_cache(9, max_seqs=1, page_size=8, max_len=72)  # more slots than the rotary tables have positions
    m.prefill_paged(_ids(64, 1), long, 0)
    with pytest.raises(Int4B200Error, match="position 65 of 64"):
        m.decode_paged(torch.zeros(1, 1, dtype=torch.long, device="cuda"), long)
    assert cache.lengths == [24, 0] and cache.lens.tolist() == [24, 0]


@torch.no_grad()
def test_score_is_the_mean_nll_of_log_softmax(hf):
    from int4_b200.decode import LlamaTP

    m = LlamaTP(hf, w4=True, max_seq=128, max_batch=2)
    ids = torch.cat([_ids(50, 7), _ids(50, 8)])
    lp, entropy, top_lp, top_ids = m.score(ids, top=3)
    ref = torch.log_softmax(m.prefill(ids, all_logits=True)[:, :-1].double(), -1)
    want = ref.gather(-1, ids[:, 1:, None])[..., 0]
    assert lp.shape == entropy.shape == (2, 49) and top_ids.shape == (2, 49, 3)
    # fp32 sums of 512 exponentials and a few roundings of numbers below 16
    assert (lp.double() - want).abs().max().item() <= 2 ** -18
    assert (entropy.double() + (ref.exp() * ref).sum(-1)).abs().max().item() <= 2 ** -17
    assert torch.equal(top_ids, torch.argsort(ref, dim=-1, descending=True, stable=True)[..., :3])
