"""Attention over 8-bit keys and values where scores are minus infinity: a row that sees keys, all of them so, is no number whatever
the context's length and the launch's form; such keys beside others have no weight; a row that sees no key gives zeros."""
import pytest
import torch

import plain_e4m3 as plain
from e4m3_cases import Cache, ragged
from llm_inference_lab_amd.cache import layout
from test_e4m3_attention_gpu import DTYPES, ops, queries, run  # noqa: F401

pytestmark = pytest.mark.gpu
FORMS = [(0, 0), (0, 1), (5, 1), (0, 2), (0, 3), (0, 4)]      # (key splits, form)


def first_numbers(cache, b, positions, code, byte=None):
    """The first number of the given keys of request ``b`` gets this code, and their scales this byte."""
    index = layout.e4m3_key_index(cache.page, cache.d)
    for p in positions:
        page, off = int(cache.table[b, p // cache.page]), p % cache.page
        if 0 <= page < cache.pages:
            cache.k.view(torch.uint8).flatten(-2)[page][:, index[off, 0]] = code
            if byte is not None:
                cache.scale[page, :, 0, off] = byte


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("splits,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [None, 5, 100])
def test_rows_whose_scores_are_all_minus_infinity(ops, d, splits, form, dtype, window):      # noqa: F811
    nq, nkv, page = 4, 2, 16
    lengths, counts = [1, 31, 32, 64, 700, 300, 90], [1, 1, 1, 2, 1, 40, 3]
    cache = Cache(lengths, nkv, d, page).fill()
    cache.table[6] = -1                                        # (sees none)
    for b, n in enumerate(lengths):
        first_numbers(cache, b, range(n), 0xb8)                # -1
    q_start, start_pos, positions, row_req = ragged(lengths, counts)
    q = queries(len(positions), nq, d, dtype, 1).view(-1, nq, d)
    plain_q = q.clone().flatten(1)
    q[:, 1, 0] = float("inf")
    q[::3, 2, 0] = float("inf")
    strange = torch.isinf(q).any(2)
    with ops.debug.force(e4m3_attention=(d, splits, form)):
        got = run(ops, cache, q.flatten(1), nq, q_start, start_pos, lengths, counts, window, 0.002).view(-1, nq, d)
        want = run(ops, cache, plain_q, nq, q_start, start_pos, lengths, counts, window, 0.002).view(-1, nq, d)
    nothing = (row_req == 6).view(-1, 1).expand_as(strange)
    assert bool(torch.isnan(got[strange & ~nothing]).all())
    assert torch.equal(got[~strange], want[~strange]) and bool(torch.isfinite(want).all())
    assert not bool(got[nothing].any()) and bool(want[~nothing].any())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("splits,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,counts", [([300], [1]), ([700], [1]), ([300], [40])])
def test_keys_beside_others(ops, d, splits, form, dtype, lengths, counts):      # noqa: F811
    """The first 128 keys have scores below float32's lowest number: what is left is the attention over the others."""
    nq, nkv, page, away = 4, 2, 16, 128
    cache = Cache(lengths, nkv, d, page).fill()
    first_numbers(cache, 0, range(lengths[0]), 0)
    first_numbers(cache, 0, range(away), 0xfe, 127)            # -448
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, dtype, 1).view(-1, nq, d)
    q[:, :, 0] = 2.0 ** 126
    with ops.debug.force(e4m3_attention=(d, splits, form)):
        got = run(ops, cache, q.flatten(1), nq, q_start, start_pos, lengths, counts, None, 0.002).double().view(-1, nq, d)
    q[:, :, 0] = 0
    for r in range(len(positions)):
        one = torch.tensor([0, 1], dtype=torch.int32)
        want, spread, reach = plain.attention(q[r:r + 1].flatten(1), nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, one,
                                              positions[r:r + 1], 1, int(positions[r]) + 1 - away, 0.002)
        tol = plain.tolerance(DTYPES[dtype], want, spread, reach, lengths[0], d)
        assert bool(((got[r:r + 1] - want).abs() <= tol).all())
