"""bfloat16 attention over 8-bit keys and values for one token or a few, up to 32 rows (tokens times heads of a group): as near to 64
bits as its outputs' own rounding allows."""
import pytest
import torch

import plain_e4m3 as plain
from e4m3_cases import Cache, ragged
from test_e4m3_attention_gpu import ops, queries, run  # noqa: F401

pytestmark = pytest.mark.gpu


def check(ops, nq, nkv, d, page, lengths, counts, window=None):      # noqa: F811
    """The float32 tolerance (scores, exponentials, sums), 2^-16 of every probability for the two bfloat16 numbers that it is taken
    as (half a step, 2^-8, of the rest that half a step left), and one rounding of the output.  Where the longest portion has more
    than 32 rows a probability is one bfloat16 number, half a step of it: 2^-8."""
    cache = Cache(lengths, nkv, d, page, seed=d).fill(d + 1)
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, "bf16", d + 2)
    got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, window, 0.002).double().view(-1, nq, d)
    want, spread, reach = plain.attention(q, nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, q_start, start_pos,
                                          len(counts), window, 0.002)
    tol = plain.tolerance(torch.float32, want, spread, reach, max(lengths), d)
    tol = tol + 2.0 ** (-16 if max(counts) * nq // nkv <= 32 else -8) * spread
    tol = tol + torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + tol)
    worst = float(((got - want).abs() / tol).max())
    assert worst <= 1.0, f"off by {worst:.3g} times the tolerance"


@pytest.mark.parametrize("nq,nkv,d,page,lengths,counts,window", [
    (14, 2, 64, 64, [700], [1], None),
    (28, 4, 128, 64, [500, 33, 2, 256], [1, 1, 1, 1], None),
    (40, 8, 128, 64, [90, 33, 5, 256], [5, 4, 5, 1], None),          # two tiles of 16 rows
    (16, 2, 64, 16, [60, 300], [4, 2], 50),
    (32, 1, 128, 16, [9, 40], [1, 1], None),                        # 32 heads to one
    (6, 2, 32, 16, [200, 3, 90], [9, 3, 1], 17),
    (3, 3, 16, 16, [20, 7], [16, 7], None),
    (5, 1, 48, 32, [33], [6], None),
    (9, 3, 96, 64, [130], [10], None),
    (8, 2, 112, 64, [30], [8], None),
    (8, 1, 256, 16, [75, 40], [2, 1], None),
])
def test_few_rows(ops, nq, nkv, d, page, lengths, counts, window):      # noqa: F811
    check(ops, nq, nkv, d, page, lengths, counts, window)


@pytest.mark.parametrize("splits", [1, 3, 40])
@pytest.mark.parametrize("counts", [[1, 1], [5, 2]])              # 7 rows, 35
def test_key_splits(ops, splits, counts):      # noqa: F811
    with ops.debug.force(e4m3_attention=(64, splits, 1)):
        check(ops, 14, 2, 64, 64, [1500, 40], counts)
