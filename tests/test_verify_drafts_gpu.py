"""The check of drafted tokens against 64-bit arithmetic, request by request (tests/plain_e4m3.py): equal tokens."""
import math

import pytest
import torch

import plain_e4m3 as plain

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from llm_inference_lab_amd.kernels.hip_ops import HipOps
    return HipOps(DEVICE)


def inputs(drafted, vocab, seed, with_draft, greedy_every=3, flat=1.0):
    gen = torch.Generator().manual_seed(seed)
    n, total = len(drafted), sum(drafted)
    rows = total + n
    logits = 3 * flat * torch.randn((rows, vocab), generator=gen)
    starts = [0]
    for k in drafted:
        starts.append(starts[-1] + k + 1)
    request = [b for b, k in enumerate(drafted) for _ in range(k)]
    at = torch.arange(total) + torch.tensor(request, dtype=torch.long)
    guess = logits[at] + flat * torch.randn((total, vocab), generator=gen)
    t = torch.tensor([0.0 if greedy_every and b % greedy_every == 1 else 0.4 + 0.3 * (b % 4) for b in range(n)])
    drafts = torch.zeros(total, dtype=torch.int32)
    for i, b in enumerate(request):
        z = guess[i] if t[b] == 0 else guess[i] / t[b] - torch.log(-torch.log(torch.rand(vocab, generator=gen).clamp(1e-9, 1 - 1e-7)))
        drafts[i] = int(z.argmax())
    uniforms = torch.randint(0, 1 << 24, (rows,), generator=gen).float() / float(1 << 24)
    return logits, guess if with_draft else None, drafts, torch.tensor(starts, dtype=torch.int32), t, uniforms


def run(ops, logits, draft, drafts, starts, t, uniforms):
    n = starts.numel() - 1
    accepted, tokens = (torch.full((n,), -9, dtype=torch.int32, device=DEVICE) for _ in range(2))
    on = [x if x is None or x.device.type == "cuda" else x.to(DEVICE) for x in (logits, draft, drafts, starts, t, uniforms)]
    ops.verify_drafts(*on, accepted, tokens)
    return accepted.tolist(), tokens.tolist()


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("drafted,vocab", [([0], 1), ([4], 5), ([1, 0, 3], 257), ([3] * 7, 4096), ([8, 0, 2, 1], 4097),
                                           ([2, 5], 50001), ([1] * 70, 1000), ([4, 4], 151936)])
def test_verify(ops, with_draft, drafted, vocab):
    for seed in range(3):
        case = inputs(drafted, vocab, seed, with_draft)
        assert run(ops, *case) == plain.verify(*case)


def test_nearly_even_distributions(ops):
    """A border every 1e-4 of the running sum, and many requests' random numbers."""
    case = inputs([2] * 60, 9001, 1, True, greedy_every=0, flat=0.2)
    assert run(ops, *case) == plain.verify(*case)


def test_random_numbers_at_the_ends(ops):
    logits, draft, drafts, starts, t, _ = inputs([2, 0, 3], 777, 5, True, greedy_every=0)
    for u in (0.0, 1.0 - 2.0 ** -24):
        case = (logits, draft, drafts, starts, t, torch.full((logits.shape[0],), u))
        assert run(ops, *case) == plain.verify(*case)


def test_ties_infinities_and_what_is_not_a_number(ops):
    for with_draft in (False, True):
        logits, draft, drafts, starts, t, u = inputs([2, 2, 2, 1, 1, 2, 0, 1, 2], 300, 7, with_draft, greedy_every=2)
        logits = logits.clone()
        logits[0, ::3] = math.nan                   # (row 0: a third of the vocabulary is no number)
        logits[3, 17] = logits[3].nan_to_num().max()   # (a tie: the smaller index)
        logits[6, :] = -math.inf                    # (no distribution)
        logits[7, :] = math.nan
        logits[8, 5:] = -math.inf                   # (few tokens have weight)
        if with_draft:
            draft = draft.clone()
            draft[1, :50] = math.nan
            draft[-1, :] = -math.inf
        drafts = drafts.clone()
        drafts[4] = 300                             # (outside the vocabulary)
        drafts[7] = -1
        case = (logits, draft, drafts, starts, t, u)
        assert run(ops, *case) == plain.verify(*case)


def test_a_draft_that_is_the_target(ops):
    """p = q: everything stands; a drafted token without weight in either falls, and p is drawn from."""
    logits, _, drafts, starts, t, u = inputs([3, 2], 500, 9, False, greedy_every=0)
    logits[1, 40] = -math.inf
    at = torch.tensor([0, 1, 2, 4, 5])
    draft = logits[at].clone()
    assert run(ops, logits, draft, drafts, starts, t, u)[0] == [3, 2]
    drafts[1] = 40
    case = (logits, draft, drafts, starts, t, u)
    got = run(ops, *case)
    assert got == plain.verify(*case) and got[0][0] == 1


def test_rows_of_a_wider_matrix(ops):
    logits, draft, drafts, starts, t, u = inputs([2, 3], 1001, 3, True)
    wide, wide_draft = torch.full((7, 1009), 99.0, device=DEVICE), torch.full((5, 1100), 99.0, device=DEVICE)
    wide[:, 3:1004], wide_draft[:, 1:1002] = logits.to(DEVICE), draft.to(DEVICE)
    got = run(ops, wide[:, 3:1004], wide_draft[:, 1:1002], drafts, starts, t, u)
    assert got == plain.verify(logits, draft, drafts, starts, t, u)


def test_the_tokens_are_the_targets(ops):
    """Over many random numbers the first token that comes out is distributed as the target's own, whatever the draft."""
    vocab, n = 6, 8192
    gen = torch.Generator().manual_seed(0)
    p, q = torch.randn(vocab, generator=gen), torch.randn(vocab, generator=gen)
    drafts = torch.multinomial(torch.softmax(q, 0), n, replacement=True, generator=gen).to(torch.int32)
    logits = p.repeat(2 * n, 1)
    starts = 2 * torch.arange(n + 1, dtype=torch.int32)
    u = torch.rand(2 * n, generator=gen)
    for draft in (q.repeat(n, 1), None):
        accepted, tokens = run(ops, logits, draft, drafts, starts, torch.ones(n), u)
        first = torch.where(torch.tensor(accepted) > 0, drafts, torch.tensor(tokens, dtype=torch.int32))
        share = torch.bincount(first.long(), minlength=vocab).double() / n
        want = torch.softmax(p.double(), 0)
        assert bool(((share - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all())      # (five standard deviations)


def test_nothing_to_verify(ops):
    empty = torch.zeros(0, dtype=torch.int32, device=DEVICE)
    none = torch.zeros(0, device=DEVICE)
    ops.verify_drafts(torch.zeros((0, 10), device=DEVICE), None, empty, torch.zeros(1, dtype=torch.int32, device=DEVICE), none,
                      none, empty, empty.clone())
    torch.cuda.synchronize()


def test_starts_that_do_not_fit(ops):
    """Row starts beyond the rows: no token for those requests, and nothing is read out of range."""
    logits, _, drafts, _, t, u = inputs([1, 1, 1], 100, 1, False)
    starts = torch.tensor([0, 2, 40, 6], dtype=torch.int32)
    accepted, tokens = run(ops, logits, None, drafts, starts, t, u)
    assert accepted[1:] == [0, 0] and tokens[1:] == [-1, -1] and tokens[0] >= 0
