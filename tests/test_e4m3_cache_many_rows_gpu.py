"""The write and the reading of 8-bit keys and values at so many rows that they go by blocks of several rows: whole words of four
keys and rows that are none, in order and out of order, with places that have no page."""
import pytest
import torch

from e4m3_cases import Cache, activations, inv_freq, ragged
from llm_inference_lab_amd.cache import layout
from test_e4m3_cache_gpu import DEVICE, DTYPES, close_queries, ops, same_cache, write_both  # noqa: F401

pytestmark = pytest.mark.gpu


def arranged(how, positions, row_req, gen):
    n = len(positions)
    if how == "shuffled":
        order = torch.randperm(n, generator=gen)
    elif how == "backwards":
        order = torch.arange(n - 1, -1, -1)
    elif how == "neighbours swapped":
        order = torch.arange(n)
        order[:n // 2 * 2] = order[:n // 2 * 2].view(-1, 2).flip(1).flatten()
    else:
        order = torch.arange(n)
    return positions[order].contiguous(), row_req[order].contiguous()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("nq,nkv,d,page,lengths,counts,how", [
    (2, 1, 16, 16, [2048], [2048], "in order"),
    (4, 2, 64, 64, [1700, 5, 801], [1642, 5, 801], "in order"),
    (3, 1, 96, 32, [2500], [2061], "in order"),                    # begins inside a word of four keys
    (3, 3, 48, 16, [1600, 500], [1600, 500], "shuffled"),
    (8, 2, 128, 64, [1900, 240], [1899, 239], "backwards"),
    (5, 1, 80, 128, [2100], [2049], "neighbours swapped"),
    (4, 16, 256, 16, [2055], [2055], "in order"),                  # codes that do not fit beside the sines
    (2, 4, 112, 64, [1] * 700 + [1430], [1] * 700 + [1430], "in order"),
    (2, 1, 128, 64, [1100], [1100], "in order"),                   # (fewer rows: a block a row)
])
def test_write(ops, dtype, nq, nkv, d, page, lengths, counts, how):      # noqa: F811
    gen = torch.Generator().manual_seed(d)
    cache = Cache(lengths, nkv, d, page)
    for b in range(len(lengths)):                                   # some places have no page
        if b % 3 == 1 or len(lengths) == 1:
            cache.table[b, (lengths[b] - 1) // page // 2] = -1
    _, _, positions, row_req = ragged(lengths, counts)
    positions, row_req = arranged(how, positions, row_req, gen)
    positions[5], row_req[6], row_req[7] = -1, -1, len(lengths)
    rows = len(positions)
    assert rows >= 1100
    qkv = activations((rows, nq + 2 * nkv, d), gen).to(DTYPES[dtype]).flatten(1)
    freq = inv_freq(d)
    dev, q, want = write_both(ops, cache, qkv, nq, freq, positions, row_req)
    same_cache(dev, cache)
    close_queries(q[8:], want[8:], DTYPES[dtype])


@pytest.mark.parametrize("nkv,d,page,how", [
    (1, 16, 16, "in order"), (3, 48, 32, "in order"), (2, 64, 64, "in order"), (5, 80, 16, "in order"), (2, 96, 128, "in order"),
    (1, 112, 64, "in order"), (8, 128, 64, "in order"), (9, 128, 64, "in order"), (5, 256, 16, "in order"), (40, 16, 16, "in order"),
    (2, 64, 64, "shuffled"), (3, 96, 16, "backwards"), (2, 128, 64, "neighbours swapped"), (1, 32, 64, "from one"),
])
@pytest.mark.parametrize("rows", [8196, 8195, 777])
def test_read(ops, nkv, d, page, how, rows):      # noqa: F811
    gen = torch.Generator().manual_seed(d + rows)
    lengths = [5200, 3, 3000]
    cache = Cache(lengths, nkv, d, page, seed=1).fill(2)
    cache.table[0, 7] = -1
    cache.table[2, 1] = cache.pages + 3
    _, _, positions, row_req = ragged(lengths, lengths)
    if how == "from one":
        positions, row_req = positions[1:], row_req[1:]
    positions, row_req = arranged(how, positions, row_req, gen)
    positions, row_req = positions[:rows].contiguous(), row_req[:rows].contiguous()
    positions[11], row_req[12], row_req[13] = -1, -1, 3
    k, v = layout.e4m3_numbers(cache.k, cache.v, cache.scale)
    where = torch.full((rows,), -1, dtype=torch.long)
    fits = (positions >= 0) & (row_req >= 0) & (row_req < 3)
    where[fits] = cache.table[row_req[fits].long(), positions[fits].long() // page].long()
    there = (where >= 0) & (where < cache.pages)
    at = where.clamp(0, cache.pages - 1)
    want_k, want_v = k[at, :, positions.long() % page], v[at, :, :, positions.long() % page]
    dev = cache.on(DEVICE)
    for out_type in DTYPES.values():
        k_out, v_out = (torch.full((rows + 1, nkv * d), 5.0, dtype=out_type, device=DEVICE) for _ in range(2))
        ops.read_kv_e4m3(dev.k, dev.v, dev.scale, nkv, d, positions.to(DEVICE), row_req.to(DEVICE), dev.table, page,
                         k_out[:rows], v_out[:rows])
        for got, want in ((k_out, want_k), (v_out, want_v)):
            assert torch.equal(got[:rows].float().cpu(), torch.where(there.view(-1, 1), want.flatten(1), 0.0))
            assert bool((got[rows:] == 5).all())


def test_nothing_stored_is_read_from_an_empty_cache(ops):      # noqa: F811
    cache = Cache([1], 2, 32, 16)
    empty = [t[:0].contiguous().to(DEVICE) for t in (cache.k, cache.v, cache.scale)]
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEVICE)
    zeros = torch.zeros(9000, dtype=torch.int32, device=DEVICE)
    for rows in (3, 9000):
        k, v = (torch.full((rows, 64), 5.0, device=DEVICE) for _ in range(2))
        ops.read_kv_e4m3(*empty, 2, 32, zeros, zeros, table, 16, k, v)
        assert not bool(k.any()) and not bool(v.any())
