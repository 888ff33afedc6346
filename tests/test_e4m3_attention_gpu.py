"""Attention over a cache of 8-bit keys and values, against 64-bit arithmetic (tests/plain_e4m3.py)."""
import math

import pytest
import torch

import plain_e4m3 as plain
from e4m3_cases import Cache, activations, ragged

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from llm_inference_lab_amd.kernels.hip_ops import HipOps
    return HipOps(DEVICE)


def queries(rows, nq, d, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (activations((rows, nq, d), gen) * 0.4).to(DTYPES[dtype]).flatten(1)


def run(ops, cache, q, nq, q_start, start_pos, lengths, counts, window, scale, n_reqs=None, dev=None, out=None):
    dev = cache.on(DEVICE) if dev is None else dev
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEVICE) if out is None else out
    ops.paged_attention_e4m3(q.to(DEVICE), nq, cache.nkv, cache.d, dev.k, dev.v, dev.scale, dev.table, cache.page,
                             q_start.to(DEVICE), start_pos.to(DEVICE), len(counts) if n_reqs is None else n_reqs,
                             max(counts), max(lengths), window, scale, out)
    return out.cpu()


def check(ops, nq, nkv, d, page, lengths, counts, dtype, window=None, seed=0, spoil=True):
    cache = Cache(lengths, nkv, d, page, seed).fill(seed + 1)
    for b, n in enumerate(lengths):                 # what lies behind the last position is not read
        if spoil:
            cache.spoil(b, range(n, -(-n // page) * page))
            if window:
                cache.spoil(b, range(0, max(0, n - counts[b] + 1 - window)))
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, dtype, seed + 2)
    scale = 1.0 / math.sqrt(d) / 64
    got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, window, scale).double().view(-1, nq, d)
    want, spread, reach = plain.attention(q, nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, q_start, start_pos,
                                          len(counts), window, scale)
    tol = plain.tolerance(DTYPES[dtype], want, spread, reach, max(lengths), d)
    worst = float(((got - want).abs() / tol).max()) if len(positions) else 0.0
    assert worst <= 1.0, f"off by {worst:.3g} times the tolerance"


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("nq,nkv,d,page,lengths,counts,window", [
    (1, 1, 16, 16, [1], [1], None),
    (14, 2, 64, 64, [700], [1], None),
    (4, 2, 64, 64, [1, 64, 65, 127, 300], [1, 1, 1, 1, 1], None),
    (28, 4, 128, 64, [500, 33, 1, 256], [1, 1, 1, 1], None),
    (28, 4, 128, 64, [500, 33, 5, 256], [5, 5, 5, 5], None),
    (5, 1, 48, 16, [100, 17], [3, 17], None),
    (16, 4, 80, 32, [90, 70], [40, 1], None),
    (9, 3, 96, 64, [130], [130], None),
    (7, 1, 112, 128, [200, 3], [9, 3], None),
    (8, 1, 256, 16, [75, 40], [1, 30], None),
    (6, 2, 32, 16, [200, 33, 90], [21, 33, 1], 17),
    (12, 2, 128, 64, [300, 300], [1, 50], 64),
    (4, 4, 64, 64, [400], [3], 1),
    (16, 2, 128, 16, [700, 300], [61, 50], 200),
    (64, 2, 64, 64, [150, 20], [1, 4], None),
    (2, 2, 128, 64, [333], [200], None),
    (14, 2, 64, 64, [290, 40], [290, 33], None),
])
def test_attention(ops, dtype, nq, nkv, d, page, lengths, counts, window):
    check(ops, nq, nkv, d, page, lengths, counts, dtype, window)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_long_histories(ops, dtype, d):
    """Few requests, many keys: the keys are split over blocks, and what they leave is put together."""
    check(ops, 4, 2, d, 64, [5003, 7], [1, 1], dtype)
    check(ops, 4, 1, d, 64, [2900], [6], dtype, window=2500)


def test_pages_that_are_not_there(ops):
    """Keys of a page that was given back, or whose number is out of range, are not seen; a row that sees none gives zeros."""
    nq, nkv, d, page = 4, 2, 64, 16
    lengths, counts = [100, 16, 40], [3, 2, 1]
    cache = Cache(lengths, nkv, d, page).fill()
    cache.table[0, 2] = -1
    cache.table[0, 4] = cache.pages + 5
    cache.table[1, 0] = -1
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(6, nq, d, "f32", 1)
    got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002).double().view(-1, nq, d)
    want, spread, reach = plain.attention(q, nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, q_start, start_pos, 3,
                                          None, 0.002)
    assert bool(((got - want).abs() <= plain.tolerance(torch.float32, want, spread, reach, 100, d)).all())
    assert not bool(got[3:5].any())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("counts", [[4], [70]])
def test_what_is_not_a_number_stays_with_the_rows_that_see_it(ops, dtype, counts):
    nq, nkv, d, page = 4, 2, 64, 16
    lengths = [100]
    cache = Cache(lengths, nkv, d, page).fill()
    cache.spoil(0, [98])
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(counts[0], nq, d, dtype, 1)
    got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002).double().view(-1, nq, d)
    assert bool(torch.isfinite(got[:-2]).all()) and bool(torch.isnan(got[-2:]).all())
    # through a window that has passed it
    got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, 1, 0.002).double().view(-1, nq, d)
    assert bool(torch.isfinite(got[:-2]).all()) and bool(torch.isnan(got[-2]).all()) and bool(torch.isfinite(got[-1]).all())
    # only one number of one value
    cache = Cache(lengths, nkv, d, page).fill()
    from llm_inference_lab_amd.cache import layout
    where = int(cache.table[0, 97 // page])
    cache.v.view(torch.uint8).flatten(-2)[where, 1, layout.e4m3_value_index(page, d)[37, 97 % page]] = 0x7f
    got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002).double().view(-1, nq, d)
    bad = torch.isnan(got)
    expect = torch.zeros_like(bad)
    expect[-3:, 2:, 37] = True
    assert torch.equal(bad, expect)


def test_requests_without_tokens_and_rows_behind_the_last(ops):
    nq, nkv, d, page = 4, 2, 64, 64
    lengths, counts = [50, 20, 30], [2, 0, 1]
    cache = Cache(lengths, nkv, d, page).fill()
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(8, nq, d, "bf16", 1)
    out = torch.full((8, nq * d), 7.0, dtype=torch.bfloat16, device=DEVICE)
    run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002, out=out)
    assert bool((out[3:] == 7).all()) and not bool((out[:3] == 7).all(1).any())
    before = out.clone()
    for n, most in ((0, 1), (3, 0)):
        ops.paged_attention_e4m3(q.to(DEVICE), nq, nkv, d, *(getattr(cache.on(DEVICE), t) for t in ("k", "v", "scale", "table")),
                                 page, q_start.to(DEVICE), start_pos.to(DEVICE), n, most, 50, None, 0.002, out)
    assert torch.equal(out, before)


def test_large_scores(ops):
    """One key far above the others, and scores far apart from step to step: the running maximum grows."""
    nq, nkv, d, page = 2, 1, 64, 64
    lengths, counts = [600], [2]
    cache = Cache(lengths, nkv, d, page).fill(exponents=(0, 8))
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    for dtype in DTYPES:
        q = queries(2, nq, d, dtype, 3)
        got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.05).double().view(-1, nq, d)
        want, spread, reach = plain.attention(q, nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, q_start, start_pos,
                                              1, None, 0.05)
        assert bool(((got - want).abs() <= plain.tolerance(DTYPES[dtype], want, spread, reach, 600, d)).all())


def test_queries_in_a_wider_matrix_on_another_stream(ops):
    nq, nkv, d, page = 4, 2, 64, 64
    lengths, counts = [90, 300], [1, 3]
    cache = Cache(lengths, nkv, d, page).fill()
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(4, nq, d, "bf16", 1)
    want = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002)
    wide = torch.cat([q, q], dim=1).to(DEVICE)
    dev = cache.on(DEVICE)
    starts, before = q_start.to(DEVICE), start_pos.to(DEVICE)
    out = torch.zeros((4, nq * d), dtype=torch.bfloat16, device=DEVICE)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.paged_attention_e4m3(wide, nq, nkv, d, dev.k, dev.v, dev.scale, dev.table, page, starts, before, 2, 3, 300, None,
                                 0.002, out)
    stream.synchronize()
    assert torch.equal(out.cpu(), want)
