"""More of the check of drafted tokens: requests of many drafts, temperatures at the ends, vocabularies of many chunks, and
single numbers that are none, against 64-bit arithmetic (tests/plain_e4m3.py)."""
import math

import pytest
import torch

import plain_e4m3 as plain
from test_verify_drafts_gpu import DEVICE, inputs, ops, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("drafted", [[15], [16], [17, 1], [31, 0, 32], [50, 33, 16]])
def test_many_drafts(ops, drafted, with_draft):      # noqa: F811
    """As many as are looked at together, one more, and several rounds of them."""
    for seed in range(3):
        case = inputs(drafted, 200, seed, with_draft)
        assert run(ops, *case) == plain.verify(*case)


@pytest.mark.parametrize("with_draft", [False, True])
def test_all_of_many_stand(ops, with_draft):      # noqa: F811
    """Nothing falls before the last round: every draft is its row's argmax by far."""
    for greedy_every in (0, 1):
        logits, draft, drafts, starts, t, u = inputs([33, 16, 17], 90, 4, with_draft, greedy_every)
        t[:] = 0.7 if greedy_every == 0 else 0.0
        place = [r for b in range(3) for r in range(int(starts[b]), int(starts[b + 1]) - 1)]
        for i, r in enumerate(place):
            logits[r, drafts[i]] = 60.0
        case = (logits, draft, drafts, starts, t, u)
        got = run(ops, *case)
        assert got == plain.verify(*case) and got[0] == [33, 16, 17]


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 30.0])
def test_temperatures(ops, temperature):      # noqa: F811
    logits, draft, drafts, starts, t, u = inputs([3, 0, 5], 5000, 2, True, greedy_every=0)
    t[:] = temperature
    for d in (draft, None):
        case = (logits, d, drafts, starts, t, u)
        assert run(ops, *case) == plain.verify(*case)


def test_a_vocabulary_of_many_chunks(ops):      # noqa: F811
    """More chunks of a row than a wave has lanes."""
    for seed in range(2):
        case = inputs([2, 1], 300007, seed, seed == 0, greedy_every=0)
        assert run(ops, *case) == plain.verify(*case)


def test_many_requests_of_many_chunks(ops):      # noqa: F811
    """More chunks of all requests than the chip holds blocks at a time; the last block of a request has one chunk less."""
    for with_draft in (False, True):
        case = inputs([1] * 62 + [0, 2], 23 * 4096 - 5, 3, with_draft, greedy_every=7)
        assert run(ops, *case) == plain.verify(*case)


def test_single_numbers_that_are_none(ops):      # noqa: F811
    """A drafted token's own logit: not a number in the draft's row (its q is zero: it stands), in the target's (its p is: it falls);
    plus infinity, of which no distribution is made."""
    logits, draft, drafts, starts, t, u = inputs([1, 1, 1, 1], 400, 11, True, greedy_every=0)
    draft[0, drafts[0]] = math.nan
    logits[2, drafts[1]] = math.nan
    logits[4, 7] = math.inf
    draft[3, 9] = math.inf
    case = (logits, draft, drafts, starts, t, u)
    got = run(ops, *case)
    assert got == plain.verify(*case)
    assert got[0] == [1, 0, 0, 0] and got[1][2:] == [-1, -1]


def test_replayed_graphs(ops):      # noqa: F811
    """One capture, replayed with new numbers in the same buffers, and eager calls between."""
    first = [x if x is None else x.to(DEVICE) for x in inputs([3, 0, 2], 9000, 1, True)]
    n = first[3].numel() - 1
    accepted, tokens = (torch.full((n,), -9, dtype=torch.int32, device=DEVICE) for _ in range(2))
    ops.verify_drafts(*first, accepted, tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(*first, accepted, tokens)
    for seed in range(4):
        case = inputs([3, 0, 2], 9000, seed, True)
        for mine, new in zip(first, case):
            mine.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert (accepted.tolist(), tokens.tolist()) == plain.verify(*case)
        assert run(ops, *case) == plain.verify(*case)
