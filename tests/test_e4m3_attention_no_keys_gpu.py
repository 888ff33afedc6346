"""Attention over 8-bit keys and values where rows see no key: a cache without pages, a block table without columns."""
import pytest
import torch

from e4m3_cases import Cache, ragged
from test_e4m3_attention_gpu import DEVICE, DTYPES, ops, queries, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("form", range(5))
@pytest.mark.parametrize("d", [16, 64, 128, 256])
def test_an_empty_cache(ops, form, d, dtype):      # noqa: F811
    """No page at all, whatever the table says, or no column in the table: the requests' rows are zeros, the others stay."""
    nq, nkv, page = 4, 2, 16
    lengths, counts = [3000, 40, 1], [1, 40, 0]
    some = Cache(lengths, nkv, d, page)
    none = some.on(DEVICE)
    none.k, none.v, none.scale = (t[:0].contiguous() for t in (none.k, none.v, none.scale))
    assert none.k.shape[0] == 0
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    rows = len(positions)
    for window in (None, 7):
        for splits in (0, 5):
            for table in (none.table, torch.full_like(none.table, -1)):
                none.table = table
                out = torch.full((rows + 2, nq * d), 7.0, dtype=DTYPES[dtype], device=DEVICE)
                with ops.debug.force(e4m3_attention=(d, splits, form)):
                    run(ops, some, queries(rows + 2, nq, d, dtype, 1), nq, q_start, start_pos, lengths, counts, window, 0.1, dev=none, out=out)
                assert not bool(out[:rows].any()) and bool((out[rows:] == 7).all())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("form", range(5))
@pytest.mark.parametrize("d", [48, 64, 128])
def test_a_table_without_columns(ops, form, d, dtype):      # noqa: F811
    nq, nkv, page = 4, 2, 16
    cache = Cache([20], nkv, d, page).fill()
    dev = cache.on(DEVICE)
    dev.table = torch.zeros((1, 0), dtype=torch.int32, device=DEVICE)
    q_start, start_pos, _, _ = ragged([20], [20])
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        out = torch.full((20, nq * d), 7.0, dtype=DTYPES[dtype], device=DEVICE)
        ops.paged_attention_e4m3(queries(20, nq, d, dtype, 1).to(DEVICE), nq, nkv, d, dev.k, dev.v, dev.scale, dev.table, page,
                                 q_start.to(DEVICE), start_pos.to(DEVICE), 1, 20, 0, None, 0.1, out)
    assert not bool(out.any())
