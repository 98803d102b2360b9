"""How the attention's tiles are cut into runs, restated in whole numbers: every tile in one run, in order, and never
more runs than the workspace has room for (7 per warp)."""
from __future__ import annotations

import random

import pytest


def deal(total, workers, shared, last):
    per = total // workers
    if shared and per >= 8 * last:
        own, longer, more = per * 5 // 8, 0, max(2 * last, per // 8)
        more_runs = (total - workers * own - last * workers + more - 1) // more
    else:
        own, longer, more, more_runs = max(per, 1), total - workers * per if per >= 1 else 0, 0, 0
    more_end = workers * own + longer + more_runs * more

    def first(r):
        if r < workers:
            return r * own + min(r, longer)
        r -= workers
        return workers * own + longer + r * more if r < more_runs else more_end + last * (r - more_runs)

    def tiles(r):
        n = own + (r < longer) if r < workers else (0 if more == 0 else (more if r < workers + more_runs else last))
        return min(n, total - first(r))

    def run_of(t):
        if t < longer * (own + 1):
            return t // (own + 1)
        if t < workers * own + longer:
            return longer + (t - longer * (own + 1)) // own
        if t < more_end:
            return workers + (t - workers * own - longer) // more
        return workers + more_runs + (t - more_end) // last

    runs = workers if more == 0 else workers + more_runs + max(0, -(-(total - more_end) // last))
    return first, tiles, run_of, runs, more


@pytest.mark.parametrize("last", [2, 4, 8])
@pytest.mark.parametrize("shared", [False, True])
def test_every_tile_is_in_one_run_in_order(shared, last):
    workers = 12
    for total in range(0, 40 * workers * last, 7):
        first, tiles, run_of, runs, _ = deal(total, workers, shared, last)
        seen = []
        for r in range(runs):
            n = tiles(r)
            if n > 0:
                assert first(r) == len(seen)
                seen += range(first(r), first(r) + n)
                assert all(run_of(t) == r for t in range(first(r), first(r) + n))
        assert seen == list(range(total))
        assert tiles(runs) <= 0 or not shared


def test_runs_fit_the_workspace_and_32_bits():
    rng = random.Random(1)
    for workers in (10, 1320, 1480):
        for last in (2, 4, 8):
            totals = [workers * 8 * last * k + d for k in range(1, 20) for d in (-1, 0, 1, workers - 1)] + [rng.randrange(1, 1 << 30) for _ in range(300)] + [1 << 30]
            for total in totals:
                first, tiles, _, runs, more = deal(total, workers, True, last)
                assert runs <= 7 * workers, (total, runs / workers)
                assert first(runs) >= total and first(workers) < 1 << 31
                if more:  # a run taken from the counter is as long as what is requested ahead, or the last one
                    short = [r for r in list(range(workers)) + [workers, runs - 2] if 0 < tiles(r) < 2]
                    assert not short
