"""Every form of the launch of attention over 8-bit keys and values, whichever the sizes would pick: the tests of
test_e4m3_attention_gpu.py with the form forced, and sizes at which a form can go wrong."""
import math

import pytest
import torch

import plain_e4m3 as plain
import test_e4m3_attention_gpu as whole
from e4m3_cases import Cache, ragged
from test_e4m3_attention_gpu import check, ops, queries, run  # noqa: F401

pytestmark = pytest.mark.gpu
FORMS = [1, 2, 3, 4]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,nkv,page,lengths,counts,window", [
    (1, 1, 16, [1], [1], None),                                    # one row, one key
    (14, 2, 64, [700], [1], None),
    (4, 2, 64, [1, 64, 65, 127, 300], [1, 1, 1, 1, 1], None),
    (28, 4, 64, [500, 33, 5, 256], [5, 5, 5, 5], None),
    (12, 2, 64, [300, 300], [1, 50], 64),
    (4, 4, 64, [400], [3], 1),
    (16, 2, 16, [700, 300], [61, 50], 200),
    (2, 2, 64, [333], [200], None),
    (14, 2, 64, [290, 40], [290, 33], None),                        # from a prompt's start, ragged
    (2, 1, 16, [16 * 300 + 5], [37], None),                         # more tiles than a wave looks up pages for at a time
    (2, 1, 16, [4700], [70], 900),
    (1, 1, 256, [513], [129], None),                                # a row past a tile of 128
])
def test_forms(ops, form, d, nq, nkv, page, lengths, counts, window):      # noqa: F811
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        check(ops, nq, nkv, d, page, lengths, counts, "bf16", window, seed=form)


@pytest.mark.parametrize("form", FORMS)
def test_what_stays_with_its_rows(ops, form):      # noqa: F811
    with ops.debug.force(e4m3_attention=(64, 0, form)):
        whole.test_pages_that_are_not_there(ops)
        for counts in ([4], [70]):
            whole.test_what_is_not_a_number_stays_with_the_rows_that_see_it(ops, "bf16", counts)
        whole.test_requests_without_tokens_and_rows_behind_the_last(ops)
        whole.test_large_scores(ops)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
def test_missing_pages_in_bfloat16(ops, form, d):      # noqa: F811
    """Whole tiles of keys without a page, the first, the last and some between; a request without any."""
    nq, nkv, page = 4, 2, 16
    lengths, counts = [700, 40, 300], [40, 40, 3]
    cache = Cache(lengths, nkv, d, page).fill()
    for slot in [0, 1, 2, 3, 4, 5, 6, 7, 8, 20, 33, 43]:
        cache.table[0, slot] = -1
    cache.table[0, 21] = cache.pages
    cache.table[1] = -1
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, "bf16", 1)
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002).double().view(-1, nq, d)
    want, spread, reach = plain.attention(q, nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page, q_start, start_pos, 3,
                                          None, 0.002)
    assert bool(((got - want).abs() <= plain.tolerance(torch.bfloat16, want, spread, reach, 700, d)).all())
    assert not bool(got[40:80].any())


@pytest.mark.parametrize("form", [0] + FORMS)
@pytest.mark.parametrize("d", [16, 32, 48, 80, 96, 112])
@pytest.mark.parametrize("nq,nkv,page,lengths,counts,window", [
    (3, 3, 16, [1, 200], [1, 200], None),
    (8, 2, 32, [300, 90, 5], [60, 33, 5], None),
    (6, 1, 64, [700], [61], 150),
])
def test_other_head_sizes(ops, form, d, nq, nkv, page, lengths, counts, window):      # noqa: F811
    """Heads that fill no 64 numbers, whose last group of values has one to three blocks; places that are no numbers."""
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        check(ops, nq, nkv, d, page, lengths, counts, "bf16", window, seed=form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [32, 48, 80, 112])
def test_one_number_that_is_none(ops, form, d):      # noqa: F811
    """A value's code in every block of its head, one after the other: only that number of the rows that see it is none."""
    from llm_inference_lab_amd.cache import layout
    nq, nkv, page = 4, 2, 16
    lengths, counts = [100], [70]
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(70, nq, d, "bf16", 1)
    for number in range(5, d, 16):
        cache = Cache(lengths, nkv, d, page).fill()
        where = int(cache.table[0, 97 // page])
        cache.v.view(torch.uint8).flatten(-2)[where, 1, layout.e4m3_value_index(page, d)[number, 97 % page]] = 0xff
        with ops.debug.force(e4m3_attention=(d, 0, form)):
            got = run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002).double().view(-1, nq, d)
        expect = torch.zeros_like(got, dtype=torch.bool)
        expect[-3:, 2:, number] = True
        assert torch.equal(torch.isnan(got), expect)


@pytest.mark.parametrize("form", [12, 22, 23, 24, 20])
@pytest.mark.parametrize("lengths,counts,window", [
    ([700, 90, 701, 300], [90, 90, 41, 90], None),
    ([200] * 64, [21, 1, 0, 33] * 16, None),                        # as many requests as are put in order; equal ones
    ([65] + [130] * 64, [33] * 65, 90),                             # one more
    ([40, 900, 33], [40, 0, 33], None),                             # the longest has no tokens
])
def test_orders_of_blocks(ops, form, lengths, counts, window):      # noqa: F811
    """By tiles, and by requests with the longest contexts first: every row once, whatever the order."""
    with ops.debug.force(e4m3_attention=(64, 0, form)):
        check(ops, 6, 2, 64, 16, lengths, counts, "bf16", window, seed=form)


@pytest.mark.parametrize("form", [0, 3, 4])
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("nq,nkv,page,lengths,counts,window", [
    (1, 1, 16, [1], [1], None),
    (4, 2, 64, [1, 64, 65, 127, 300], [1, 1, 1, 65, 1], None),
    (12, 2, 64, [300, 300], [1, 50], 64),
    (4, 4, 64, [400], [3], 1),
    (2, 1, 16, [16 * 300 + 5], [37], None),                         # more tiles than a wave looks up pages for at a time
    (16, 2, 16, [700, 300], [129, 50], 200),
])
def test_forms_in_float32(ops, form, d, nq, nkv, page, lengths, counts, window):      # noqa: F811
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        check(ops, nq, nkv, d, page, lengths, counts, "f32", window, seed=form)


@pytest.mark.parametrize("form", [3, 4])
def test_what_stays_with_its_rows_in_float32(ops, form):      # noqa: F811
    with ops.debug.force(e4m3_attention=(64, 0, form)):
        for counts in ([4], [70]):
            whole.test_what_is_not_a_number_stays_with_the_rows_that_see_it(ops, "f32", counts)


@pytest.mark.parametrize("form", [13, 14, 23, 24])
def test_orders_of_blocks_in_float32(ops, form):      # noqa: F811
    with ops.debug.force(e4m3_attention=(128, 0, form)):
        check(ops, 6, 2, 128, 16, [700, 90, 701, 300], [90, 90, 41, 90], "f32", None, seed=form)


def test_many_float32_rows(ops):      # noqa: F811
    """As many as take the codes staged in LDS without a form forced; the same bits every time."""
    nq, nkv, d, page = 32, 4, 128, 64
    lengths, counts = [260, 400, 300, 260], [256, 200, 256, 33]
    check(ops, nq, nkv, d, page, lengths, counts, "f32", None, seed=3)
    cache = Cache(lengths, nkv, d, page).fill()
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, "f32", 1)
    dev = cache.on(whole.DEVICE)
    outs = [run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002, dev=dev) for _ in range(3)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("splits", [1, 2, 7, 64])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_key_splits(ops, splits, dtype):      # noqa: F811
    """Splits that leave some blocks without a key."""
    with ops.debug.force(e4m3_attention=(64, splits, 1)):
        check(ops, 14, 2, 64, 64, [700, 3, 90], [1, 1, 2], dtype)
        check(ops, 4, 2, 64, 16, [700, 30], [20, 11], dtype, window=100)


@pytest.mark.parametrize("form", FORMS)
def test_the_same_every_time(ops, form):      # noqa: F811
    """Sums are taken in one order: the same bits from every run."""
    nq, nkv, d, page = 28, 4, 128, 64
    lengths, counts = [1500, 700, 1100], [90, 200, 1]
    cache = Cache(lengths, nkv, d, page).fill()
    q_start, start_pos, positions, _ = ragged(lengths, counts)
    q = queries(len(positions), nq, d, "bf16", 1)
    dev = cache.on(whole.DEVICE)
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        outs = [run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 1 / math.sqrt(d) / 64, dev=dev) for _ in range(4)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("form", [0] + FORMS)
def test_positions_beyond_the_table(ops, form):      # noqa: F811
    """Rows far behind what the table has room for see what it has, and no walk goes further."""
    nq, nkv, d, page = 4, 2, 64, 16
    cache = Cache([80], nkv, d, page).fill()
    q = queries(33, nq, d, "bf16", 1)
    far = torch.tensor([1 << 30], dtype=torch.int32)
    with ops.debug.force(e4m3_attention=(d, 0, form)):
        got = run(ops, cache, q, nq, torch.tensor([0, 33], dtype=torch.int32), far, [80], [33], None, 0.002)
        gone = run(ops, cache, q, nq, torch.tensor([0, 33], dtype=torch.int32), far, [80], [33], 50, 0.002)
    one = torch.tensor([79], dtype=torch.int32)
    for i in (0, 17, 32):
        want, spread, reach = plain.attention(q[i:i + 1], nq, nkv, d, cache.k, cache.v, cache.scale, cache.table, page,
                                              torch.tensor([0, 1], dtype=torch.int32), one, 1, None, 0.002)
        tol = plain.tolerance(torch.bfloat16, want, spread, reach, 80, d)
        assert bool(((got[i].double().view(1, nq, d) - want).abs() <= tol).all())
    assert not bool(gone.any())
