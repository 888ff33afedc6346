"""The write of 8-bit keys and values and their reading, against 64-bit arithmetic (tests/plain_e4m3.py)."""
import math

import pytest
import torch

import plain_e4m3 as plain
from e4m3_cases import Cache, activations, inv_freq, ragged

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from llm_inference_lab_amd.kernels.hip_ops import HipOps
    return HipOps(DEVICE)


def write_both(ops, cache, qkv, nq, freq, positions, row_req, q_out=None):
    """Stores with the kernel and plainly; (the kernel's cache, the plain one's, queries, plain queries)."""
    rows, nkv, d = qkv.shape[0], cache.nkv, cache.d
    dev = cache.on(DEVICE)
    x = qkv.to(DEVICE)
    q = torch.full((rows, nq * d), 7.0, dtype=qkv.dtype, device=DEVICE) if q_out is None else q_out(x)
    ops.rope_kv_write_e4m3(x, nq, nkv, d, None if freq is None else freq.to(DEVICE), positions.to(DEVICE),
                           row_req.to(DEVICE), dev.table, cache.page, dev.k, dev.v, dev.scale, q)
    want = plain.write(qkv, nq, nkv, d, freq, positions, row_req, cache.table, cache.page, cache.k, cache.v, cache.scale)
    return dev, q.cpu().double(), want


def same_cache(dev, cache):
    for name in ("scale", "k", "v"):
        got, want = getattr(dev, name).view(torch.uint8).cpu(), getattr(cache, name).view(torch.uint8)
        differ = (got != want).nonzero()[:6].tolist()
        assert not differ, f"{name}: " + ", ".join(f"{at}: {int(got[tuple(at)])} != {int(want[tuple(at)])}" for at in differ)


def close_queries(got, want, dtype):
    half = torch.finfo(dtype).eps / 2 + torch.finfo(torch.float32).eps      # one rounding, behind one to 32 bits
    assert bool(((got - want).abs() <= half * want.abs() + 1e-37).all())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("nq,nkv,d,page,lengths,counts", [
    (2, 1, 16, 16, [1], [1]),
    (4, 2, 64, 64, [700, 5, 64], [1, 1, 1]),
    (4, 4, 48, 16, [33, 17, 1], [33, 2, 1]),
    (6, 2, 32, 32, [40, 100], [37, 21]),
    (5, 1, 80, 128, [300], [77]),
    (7, 1, 112, 64, [65, 66], [2, 60]),
    (8, 2, 128, 64, [130, 31000, 63], [129, 3, 1]),
    (4, 2, 256, 16, [50], [19]),
])
def test_write_and_read(ops, dtype, nq, nkv, d, page, lengths, counts):
    gen = torch.Generator().manual_seed(d + len(lengths))
    cache = Cache(lengths, nkv, d, page)
    _, _, positions, row_req = ragged(lengths, counts)
    rows = len(positions)
    qkv = activations((rows, nq + 2 * nkv, d), gen).to(DTYPES[dtype]).flatten(1)
    dev, q, want = write_both(ops, cache, qkv, nq, inv_freq(d), positions, row_req)
    same_cache(dev, cache)
    close_queries(q, want, DTYPES[dtype])
    # and back, in both types, in another order
    order = torch.randperm(rows, generator=gen)
    for out_type in DTYPES.values():
        k, v = (torch.full((rows, nkv * d), 5.0, dtype=out_type, device=DEVICE) for _ in range(2))
        ops.read_kv_e4m3(dev.k, dev.v, dev.scale, nkv, d, positions[order].to(DEVICE), row_req[order].to(DEVICE), dev.table,
                         page, k, v)
        for i, r in enumerate(order.tolist()):
            wk, wv = plain.stored(cache.k, cache.v, cache.scale, cache.table, int(row_req[r]), int(positions[r]), page)
            assert torch.equal(k[i].cpu().double(), wk.flatten()) and torch.equal(v[i].cpu().double(), wv.flatten())


def test_without_a_rotation_and_in_place(ops):
    nq, nkv, d, page = 4, 2, 64, 16
    gen = torch.Generator().manual_seed(3)
    lengths, counts = [40, 20], [9, 20]
    _, _, positions, row_req = ragged(lengths, counts)
    qkv = activations((29, nq + 2 * nkv, d), gen).to(torch.bfloat16).flatten(1)
    cache = Cache(lengths, nkv, d, page)
    dev, q, want = write_both(ops, cache, qkv, nq, None, positions, row_req)
    same_cache(dev, cache)
    assert torch.equal(q, qkv.double()[:, :nq * d])
    # turned, the queries written over the projections' own columns
    cache = Cache(lengths, nkv, d, page)
    dev, q, want = write_both(ops, cache, qkv, nq, inv_freq(d), positions, row_req, q_out=lambda x: x[:, :nq * d])
    same_cache(dev, cache)
    close_queries(q, want, torch.bfloat16)


def test_rows_of_a_wider_matrix(ops):
    """Projections and queries that are columns of wider matrices; an odd row stride."""
    nq, nkv, d, page = 2, 1, 32, 16
    gen = torch.Generator().manual_seed(4)
    wide = activations((11, nq + 2 * nkv + 2, d), gen).to(torch.bfloat16).flatten(1)
    wide = torch.cat([wide, wide[:, :5]], dim=1).contiguous()
    _, _, positions, row_req = ragged([11], [11])
    cache = Cache([11], nkv, d, page)
    dev = cache.on(DEVICE)
    x = wide.to(DEVICE)[:, 3:3 + (nq + 2 * nkv) * d]
    q_wide = torch.full((11, nq * d + 9), 7.0, dtype=torch.bfloat16, device=DEVICE)
    ops.rope_kv_write_e4m3(x, nq, nkv, d, inv_freq(d).to(DEVICE), positions.to(DEVICE), row_req.to(DEVICE), dev.table, page,
                           dev.k, dev.v, dev.scale, q_wide[:, 1:1 + nq * d])
    want = plain.write(x.cpu(), nq, nkv, d, inv_freq(d), positions, row_req, cache.table, page, cache.k, cache.v, cache.scale)
    same_cache(dev, cache)
    close_queries(q_wide[:, 1:1 + nq * d].cpu().double(), want, torch.bfloat16)
    assert bool((q_wide[:, :1] == 7).all()) and bool((q_wide[:, 1 + nq * d:] == 7).all())


def test_positions_without_a_page(ops):
    """A page that was given back, a page number out of range, a position behind the table, a negative one, a request
    that is not there: nothing is stored, zeros are read, and the others are as ever."""
    nq, nkv, d, page = 2, 2, 32, 16
    gen = torch.Generator().manual_seed(5)
    cache = Cache([64, 64], nkv, d, page)
    cache.table[0, 1] = -1
    cache.table[1, 2] = cache.pages
    positions = torch.tensor([0, 17, 63, 64, -1, 40, 3, 8], dtype=torch.int32)
    row_req = torch.tensor([0, 0, 0, 0, 0, 1, 2, 1], dtype=torch.int32)
    qkv = activations((8, nq + 2 * nkv, d), gen).flatten(1)
    dev, q, want = write_both(ops, cache, qkv, nq, inv_freq(d), positions, row_req)
    same_cache(dev, cache)
    close_queries(q, want, torch.float32)
    k, v = (torch.full((8, nkv * d), 5.0, device=DEVICE) for _ in range(2))
    ops.read_kv_e4m3(dev.k, dev.v, dev.scale, nkv, d, positions.to(DEVICE), row_req.to(DEVICE), dev.table, page, k, v)
    for r in (1, 3, 4, 5, 6):
        assert not bool(k[r].any()) and not bool(v[r].any())
    for r in (0, 2, 7):
        wk, _ = plain.stored(cache.k, cache.v, cache.scale, cache.table, int(row_req[r]), int(positions[r]), page)
        assert torch.equal(k[r].cpu().double(), wk.flatten())


def test_numbers_at_the_borders(ops):
    """Zeros, one number alone, the largest and the smallest, ties, infinities and what is not a number."""
    nq, nkv, d, page = 1, 1, 32, 16
    rows = [torch.zeros(d), torch.full((d,), 448.0), torch.full((d,), 448.0 * (1 + 2.0 ** -23)), torch.full((d,), 1e-38),
            torch.full((d,), 3.38e38), torch.full((d,), 2.0 ** -109), torch.full((d,), 2.0 ** -110), torch.full((d,), -0.0)]
    x = torch.linspace(-440, 440, d)
    x[0], x[1], x[2] = math.inf, -math.inf, math.nan
    rows.append(x)
    rows.append(torch.full((d,), math.nan))
    ties = torch.tensor([1.0625, 1.1875, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 448.0]).repeat(4)
    rows += [ties, -ties * 8, ties * 2.0 ** -60]
    stored = torch.stack(rows)
    for r, row in enumerate(rows):                        # one number next to a border between two codes, either side
        near = ties * (1 + (2.0 ** -23 if r % 2 else -2.0 ** -23))
        near[7] = 448.0
        stored = torch.cat([stored, near.view(1, -1)])
    n = stored.shape[0]
    qkv = torch.cat([torch.ones((n, nq * d)), stored, stored.flip(1)], dim=1)
    _, _, positions, row_req = ragged([n], [n])
    cache = Cache([n], nkv, d, page)
    dev, q, _ = write_both(ops, cache, qkv, nq, None, positions, row_req)
    same_cache(dev, cache)


def test_far_positions(ops):
    """Angles in 64 bits: a turn of a position near 2^31 (the table's pages only where they are needed)."""
    nq, nkv, d, page = 1, 1, 16, 16
    gen = torch.Generator().manual_seed(6)
    far = 1 << 20
    cache = Cache([16], nkv, d, page)
    cache.table = torch.full((1, far // page + 1), -1, dtype=torch.int32)
    cache.table[0, far // page] = 1
    qkv = activations((3, nq + 2 * nkv, d), gen).flatten(1)
    positions = torch.tensor([far, far + 5, 2 ** 31 - 1], dtype=torch.int32)
    dev, q, want = write_both(ops, cache, qkv, nq, inv_freq(d), positions, torch.zeros(3, dtype=torch.int32))
    same_cache(dev, cache)
    # (a sine of 2^31 is known to the rounding of its angle: 2^31 * 2^-53)
    assert bool(((q - want).abs() <= 2.0 ** -20 * want.abs() + 2.0 ** -21).all())
    close_queries(q[:2], want[:2], torch.float32)


def test_no_rows(ops):
    cache = Cache([16], 1, 16, 16).on(DEVICE)
    empty = torch.zeros((0, 48), device=DEVICE)
    none = torch.zeros(0, dtype=torch.int32, device=DEVICE)
    ops.rope_kv_write_e4m3(empty, 1, 1, 16, None, none, none, cache.table, 16, cache.k, cache.v, cache.scale, empty[:, :16])
    ops.read_kv_e4m3(cache.k, cache.v, cache.scale, 1, 16, none, none, cache.table, 16, empty[:, :16].contiguous(),
                     empty[:, :16].contiguous())
    torch.cuda.synchronize()
