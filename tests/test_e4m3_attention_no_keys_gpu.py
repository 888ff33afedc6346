"""Attention over 8-bit keys and values where rows see no key: a cache without pages, a block table without columns,
and missing pages in whose place nothing of what lies in the first page gets through."""
import pytest
import torch

import plain_e4m3 as plain
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


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("form", range(5))
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("window", [None, 90])
def test_the_first_page_in_a_missing_ones_place(ops, form, d, dtype, window):      # noqa: F811
    """Every place that no request has holds codes that are not numbers and bytes of 255, the first page among them."""
    nq, nkv, page = 4, 2, 16
    lengths, counts = [700, 40, 300], [40, 40, 3]
    cache = Cache(lengths, nkv, d, page).fill()
    first = (cache.table == 0).nonzero()
    if len(first):                                  # (the request that has page 0 gives it back)
        cache.table[tuple(first[0])] = -1
    for slot in [0, 1, 2, 3, 4, 5, 6, 7, 8, 20, 33, 43]:
        cache.table[0, slot] = -1
    cache.table[0, 21] = cache.pages
    cache.table[1] = -1
    taken = set(cache.table.flatten().tolist())
    spare = [p for p in range(cache.pages) if p not in taken]
    assert 0 in spare
    for t, byte in ((cache.k, 0x7f), (cache.v, 0xff), (cache.scale, 0xff)):
        t.view(torch.uint8)[spare] = byte
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, dtype, 1)
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, window, 0.002).double().view(-1, nq, d)
    want, spread, reach = plain.attention(q, nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, q_start, start_pos, 3,
                                          window, 0.002)
    assert bool(((got - want).abs() <= plain.tolerance(DTYPES[dtype], want, spread, reach, 700, d)).all())
    assert not bool(got[40:80].any())
