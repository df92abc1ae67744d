"""Beam steps of many groups and rows: clusters of four, two and no CTAs that join a group, and more slices of rows than CTAs that run at a time."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops
from test_beam_step_gpu import BF16, F32, check, inputs


def odd(logits, by):
    """The same rows, beginning ``by`` elements behind a row's start in memory of an odd width."""
    wide = torch.full((logits.shape[0], logits.shape[1] + by + 2), math.nan, dtype=logits.dtype, device="cuda")
    wide[:, by:by + logits.shape[1]] = logits
    return wide[:, by:by + logits.shape[1]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [74, 75, 80, 148, 149, 160, 296, 297, 320])
def test_groups_of_which_some_need_64_bits(dtype, groups):
    """Rows of every third group are the same, so that sums in 64 bits decide; the groups beside them have none of that."""
    n, V = 3, 301
    logits, scores, g = inputs(groups, n, V, dtype, seed=groups)
    logits.view(groups, n, V)[::3] = logits.view(groups, n, V)[::3, :1]
    scores[::3] = scores[::3, :1]
    check(logits, scores)
    check(odd(logits, 1), scores, 7)
    finished = torch.rand(groups, n, generator=g) < 0.3
    check(odd(logits, 3), scores, 4, finished)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups,n,V", [(200, 4, 257), (700, 1, 300), (40, 16, 4100), (4, 16, 50304), (2, 32, 50301)])
def test_more_slices_than_run_at_a_time(dtype, groups, n, V):
    """CTAs send for the slice behind theirs: rows that begin at any element, the next row finished or without a score."""
    logits, scores, g = inputs(groups, n, V, dtype, seed=V)
    finished = torch.rand(groups, n, generator=g) < 0.3
    scores[torch.rand(groups, n, generator=g).cuda() < 0.1] = -math.inf
    for by in (0, 1, 5):
        check(odd(logits, by) if by else logits, scores, min(n, 5), finished)


def test_many_groups_in_two_streams_at_a_time():
    logits, scores, _ = inputs(160, 4, 2500, BF16)
    other, other_scores, _ = inputs(80, 8, 2500, BF16, seed=1)
    want = [ops.beam_step(logits, scores), ops.beam_step(other, other_scores)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, args in enumerate(((logits, scores), (other, other_scores))):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.beam_step(*args))
    torch.cuda.synchronize()
    for w, calls in zip(want, got):
        for c in calls:
            assert all(torch.equal(a, b) for a, b in zip(w, c))
