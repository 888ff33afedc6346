"""Pages whose bytes lie beyond 2^32, and key splits in a captured graph."""
import pytest
import torch

from e4m3_cases import Cache, activations, inv_freq, ragged
from test_e4m3_attention_gpu import DEVICE, DTYPES, ops, queries, run  # noqa: F401

pytestmark = pytest.mark.gpu


def test_pages_beyond_32_bits(ops):      # noqa: F811
    """The same rows written to low pages and to the last ones of 4.7 GB of keys and as many of values: the same bytes, the same
    numbers read back, the same attention."""
    nkv, d, page, nq = 8, 128, 64, 16
    pages = 72000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not the memory for it")
    k = torch.zeros((pages, nkv, page, d), dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn)
    v = torch.zeros((pages, nkv, d, page), dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn)
    scale = torch.zeros((pages, nkv, 2, page), dtype=torch.uint8, device=DEVICE)
    assert k.numel() > 1 << 32
    length, need = 2100, 33
    low = torch.arange(need, dtype=torch.int32)
    table = torch.stack([low, pages - 1 - low]).to(DEVICE)
    gen = torch.Generator().manual_seed(0)
    row = activations((length, nq + 2 * nkv, d), gen).to(torch.bfloat16).flatten(1)
    qkv = torch.cat([row, row]).to(DEVICE)
    positions = torch.arange(length, dtype=torch.int32, device=DEVICE).repeat(2)
    row_req = torch.arange(2, dtype=torch.int32, device=DEVICE).repeat_interleave(length)
    q = torch.empty((2 * length, nq * d), dtype=torch.bfloat16, device=DEVICE)
    ops.rope_kv_write_e4m3(qkv, nq, nkv, d, inv_freq(d).to(DEVICE), positions, row_req, table, page, k, v, scale, q)
    for t in (k.view(torch.uint8), v.view(torch.uint8), scale):
        assert torch.equal(t[:need], t[pages - need:].flip(0)) and bool(t[:need].any())
    got = torch.empty((2, 2 * length, nkv * d), dtype=torch.bfloat16, device=DEVICE)
    for rows in (2 * length, 9):
        ops.read_kv_e4m3(k, v, scale, nkv, d, positions[-rows:], row_req[-rows:], table, page, got[0, :rows], got[1, :rows])
        if rows == 2 * length:
            assert torch.equal(got[:, :length], got[:, length:]) and bool(got.any())
    start_pos = torch.tensor([length - 40, length - 40], dtype=torch.int32, device=DEVICE)
    q_start = torch.tensor([0, 40, 80], dtype=torch.int32, device=DEVICE)
    for form in range(5):
        for dtype in DTYPES.values() if form < 2 else (torch.bfloat16,):
            x = torch.cat([q[length - 40:length]] * 2).to(dtype)
            out = torch.empty_like(x)
            with ops.debug.force(e4m3_attention=(d, 0, form)):
                ops.paged_attention_e4m3(x, nq, nkv, d, k, v, scale, table, page, q_start, start_pos, 2, 40, length, None, 0.01, out)
            assert torch.equal(out[:40], out[40:]) and bool(torch.isfinite(out).all()) and bool(out.any())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_key_splits_in_a_graph(ops, dtype):      # noqa: F811
    """One capture with splits that meet in the workspace, replayed over new queries and lengths with eager calls between."""
    nq, nkv, d, page = 14, 2, 64, 64
    lengths, counts = [4000, 2500, 700], [1, 1, 1]
    cache = Cache(lengths, nkv, d, page).fill()
    dev = cache.on(DEVICE)
    q_start, start_pos, _, _ = ragged(lengths, counts)
    q_start, start_pos = q_start.to(DEVICE), start_pos.to(DEVICE)
    q = queries(3, nq, d, dtype, 0).to(DEVICE)
    out = torch.zeros_like(q)

    def step(x, at, y):
        ops.paged_attention_e4m3(x, nq, nkv, d, dev.k, dev.v, dev.scale, dev.table, page, q_start, at, 3, 1, 4000, None, 0.002, y)

    step(q, start_pos, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, start_pos, out)
    for turn in range(6):
        fresh = queries(3, nq, d, dtype, turn + 1).to(DEVICE)
        at = torch.tensor([3999 - 100 * turn, 2499 - 400 * turn, 699 - turn], dtype=torch.int32, device=DEVICE)
        q.copy_(fresh)
        start_pos.copy_(at)
        out.fill_(5)
        graph.replay()
        again = torch.empty_like(out)
        step(fresh, at, again)
        ops.workspace.fill_(float("nan"))
        torch.cuda.synchronize()
        assert torch.equal(out, again)


def test_queries_at_the_least_stride_and_place(ops):      # noqa: F811
    """float32 queries whose rows are 4 numbers apart from a multiple of 8, bfloat16 ones 8: what 16-byte loads can take."""
    nq, nkv, d, page = 4, 2, 64, 64
    lengths, counts = [90, 300], [1, 40]
    cache = Cache(lengths, nkv, d, page).fill()
    q_start, start_pos, _, _ = ragged(lengths, counts)
    for dtype, more in (("f32", 4), ("bf16", 8)):
        q = queries(41, nq, d, dtype, 1)
        wide = torch.zeros((41, nq * d + more), dtype=DTYPES[dtype])
        wide[:, more:] = q
        dev = cache.on(DEVICE)
        out = torch.zeros((41, nq * d), dtype=DTYPES[dtype], device=DEVICE)
        ops.paged_attention_e4m3(wide.to(DEVICE)[:, more:], nq, nkv, d, dev.k, dev.v, dev.scale, dev.table, page, q_start.to(DEVICE),
                                 start_pos.to(DEVICE), 2, 40, 300, None, 0.002, out)
        assert torch.equal(out.cpu(), run(ops, cache, q, nq, q_start, start_pos, lengths, counts, None, 0.002))
