"""Attention over 8-bit keys and values by key splits: the launch that puts the splits together writes the rows that the first one
has sums of and no others, as one launch does."""
import pytest
import torch

from e4m3_cases import Cache
from test_e4m3_attention_gpu import DEVICE, DTYPES, ops, queries  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("starts,most,written", [
    ([0, 2, 12], 10, [0, 1]),                       # the second request has more rows than there are
    ([2, 3, 5], 2, [2, 3, 4]),                      # rows of no request in front of the first and behind the last
    ([-2, 1, 3], 3, [1, 2]),                        # a request in front of the rows
    ([0, 9, 4, 6], 9, [4, 5]),                      # a start past the rows: neither its request nor the one before fits
    ([0, 3, 3, 5], 3, [0, 1, 2, 3, 4]),
    ([0, 70, 72], 1, None),                         # more tokens than the call says: the launch's tiles, and no further
])
def test_rows_that_are_written(ops, dtype, starts, most, written):      # noqa: F811
    nq, nkv, d, page = 6, 3, 64, 16
    rows = 8 if written is not None else 80
    lengths = [500, 400, 300][:len(starts) - 1]
    cache = Cache(lengths, nkv, d, page).fill()
    dev = cache.on(DEVICE)
    q = queries(rows, nq, d, dtype, 1).to(DEVICE)
    q_start = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    start_pos = torch.tensor([n - 90 for n in lengths], dtype=torch.int32, device=DEVICE)
    outs = []
    for splits in (1, 5):
        ops.workspace.fill_(float("nan"))           # (what a call before this one may have left)
        out = torch.full((rows, nq * d), 7.0, dtype=DTYPES[dtype], device=DEVICE)
        with ops.debug.force(e4m3_attention=(d, splits, 1)):
            ops.paged_attention_e4m3(q, nq, nkv, d, dev.k, dev.v, dev.scale, dev.table, page, q_start, start_pos, len(lengths), most,
                                     max(lengths), None, 0.002, out)
        outs.append(out.float().cpu())
    left = [(out == 7).all(1).nonzero().flatten().tolist() for out in outs]
    assert left[0] == left[1] and all(bool(torch.isfinite(out).all()) for out in outs)
    if written is not None:
        assert left[0] == [r for r in range(rows) if r not in written]
    else:
        assert 9 <= len(left[0]) < 80
