"""The operators of the 8-bit cache and the check of drafted tokens together, as a serving loop uses them: a one-layer
model decodes with drafted tokens and without, from the same pages."""
import math

import pytest
import torch

import plain_e4m3 as plain
from e4m3_cases import Cache, inv_freq

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
NQ, NKV, D, PAGE, VOCAB = 4, 2, 64, 16, 300


@pytest.fixture(scope="module")
def ops():
    from llm_inference_lab_amd.kernels.hip_ops import HipOps
    return HipOps(DEVICE)


class Model:
    """Token -> embedding -> attention over the cache -> logits, in float32; random weights."""

    def __init__(self, ops, requests, room, seed=0, dtype=torch.float32):
        gen = torch.Generator().manual_seed(seed)
        hidden = NQ * D

        def w(*shape):
            return (torch.randn(shape, generator=gen) / math.sqrt(shape[0])).to(DEVICE)
        self.ops, self.dtype = ops, dtype
        self.embed, self.qkv, self.out = w(VOCAB, hidden) * math.sqrt(VOCAB), w(hidden, (NQ + 2 * NKV) * D) * 1.5, w(hidden, VOCAB) * 2
        self.freq = inv_freq(D).to(DEVICE)
        self.room = room
        self.host = Cache([room] * requests, NKV, D, PAGE, seed)
        self.cache = self.host.on(DEVICE)

    def step(self, tokens, before):
        """Logits of every row; ``tokens[b]`` are request b's new tokens, ``before[b]`` what it has stored."""
        rows = sum(len(t) for t in tokens)
        starts = [0]
        for t in tokens:
            starts.append(starts[-1] + len(t))
        i32 = dict(dtype=torch.int32, device=DEVICE)
        positions = torch.tensor([n + j for t, n in zip(tokens, before) for j in range(len(t))], **i32)
        row_req = torch.tensor([b for b, t in enumerate(tokens) for _ in t], **i32)
        x = self.embed[torch.tensor([t for ts in tokens for t in ts], device=DEVICE)]
        qkv = (x @ self.qkv).to(self.dtype)
        q = qkv[:, :NQ * D]
        c, ops = self.cache, self.ops
        ops.rope_kv_write_e4m3(qkv, NQ, NKV, D, self.freq, positions, row_req, c.table, PAGE, c.k, c.v, c.scale, q)
        out = torch.empty((rows, NQ * D), dtype=self.dtype, device=DEVICE)
        longest = max(n + len(t) for t, n in zip(tokens, before))
        ops.paged_attention_e4m3(q, NQ, NKV, D, c.k, c.v, c.scale, c.table, PAGE, torch.tensor(starts, **i32),
                                 torch.tensor(before, **i32), len(tokens), max(map(len, tokens)), longest, None, 1 / math.sqrt(D), out)
        return (x + out.float()) @ self.out, starts


def decode(model, prompts, count, drafter, temperature, seed):
    """``count`` tokens or more of every request; ``drafter(b, so_far)`` gives drafted tokens (and their logits or None)."""
    ops, n = model.ops, len(prompts)
    gen = torch.Generator().manual_seed(seed)
    so_far, stored = [[] for _ in prompts], [0] * n
    pending = [list(p) for p in prompts]
    accepted, tokens = (torch.empty(n, dtype=torch.int32, device=DEVICE) for _ in range(2))
    temperatures = torch.full((n,), temperature, device=DEVICE)
    steps = 0
    while min(len(s) for s in so_far) < count:
        drafted = [drafter(b, so_far[b]) if so_far[b] else [] for b in range(n)]
        logits, starts = model.step([p + d for p, d in zip(pending, drafted)], stored)
        keep = [r for b in range(n) for r in range(starts[b + 1] - len(drafted[b]) - 1, starts[b + 1])]
        row_start = [0]
        for d in drafted:
            row_start.append(row_start[-1] + len(d) + 1)
        uniforms = torch.rand(len(keep), generator=gen).to(DEVICE)
        ops.verify_drafts(logits[keep], None, torch.tensor([t for d in drafted for t in d], dtype=torch.int32, device=DEVICE),
                          torch.tensor(row_start, dtype=torch.int32, device=DEVICE), temperatures, uniforms, accepted, tokens)
        for b, (k, token) in enumerate(zip(accepted.tolist(), tokens.tolist())):
            stored[b] += len(pending[b]) + k           # (what fell is written over by the next step)
            so_far[b] += drafted[b][:k] + [token]
            pending[b] = [token]
        steps += 1
    return [s[:count] for s in so_far], steps


PROMPTS = [[5, 9, 200, 7], [17] * 40, [3]]


def test_drafts_change_no_greedy_token(ops):
    plain_tokens, steps = decode(Model(ops, 3, 128), PROMPTS, 40, lambda b, s: [], 0.0, 1)
    assert steps == 40

    def sometimes_right(b, s):
        right = plain_tokens[b][len(s):len(s) + 3]
        return [t if (len(s) + j + b) % 4 else (t + 1) % VOCAB for j, t in enumerate(right)]
    tokens, steps = decode(Model(ops, 3, 128), PROMPTS, 40, sometimes_right, 0.0, 2)
    assert tokens == plain_tokens and steps < 30


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampled_runs_repeat(ops, dtype):
    """The same random numbers, the same tokens; and the cache holds what was written last."""
    def drafter(b, s):
        return [(s[-1] * 7 + 3) % VOCAB, (s[-1] + b) % VOCAB]
    first = Model(ops, 3, 128, dtype=dtype)
    runs = [decode(first, PROMPTS, 25, drafter, 0.8, 5), decode(Model(ops, 3, 128, dtype=dtype), PROMPTS, 25, drafter, 0.8, 5)]
    assert runs[0] == runs[1]
    positions = torch.arange(20, dtype=torch.int32, device=DEVICE)
    row_req = torch.ones(20, dtype=torch.int32, device=DEVICE)
    c = first.cache
    k, v = (torch.empty((20, NKV * D), device=DEVICE) for _ in range(2))
    ops.read_kv_e4m3(c.k, c.v, c.scale, NKV, D, positions, row_req, c.table, PAGE, k, v)
    host = [t.cpu() for t in (c.k, c.v, c.scale, c.table)]
    for p in range(20):
        want = plain.stored(*host, 1, p, PAGE)
        assert torch.equal(k[p].cpu().double().view(NKV, D), want[0]) and torch.equal(v[p].cpu().double().view(NKV, D), want[1])
    qkv = (first.embed[torch.tensor(PROMPTS[1][:20], device=DEVICE)] @ first.qkv).to(dtype).double().view(20, -1, D)
    value = qkv[:, NQ + NKV:].flatten(1).cpu()
    # (a value's scale is at most 2 / 448 of its largest number, and e4m3 rounds by 2^-4 of a number or half a step of 2^-9 scales)
    largest = value.view(20, NKV, D).abs().amax(-1, keepdim=True).expand(-1, -1, D).flatten(1)
    assert bool(((v.cpu().double() - value).abs() <= value.abs() / 16 + largest * (2 / 448) / 1024).all())


def test_a_captured_step_replays(ops):
    """Write, attention and check in one graph, replayed over growing contexts with eager work between."""
    n, drafts = 3, 2
    rows = n * (drafts + 1)
    i32 = dict(dtype=torch.int32, device=DEVICE)
    gen = torch.Generator().manual_seed(3)
    cache = Cache([200] * n, NKV, D, PAGE).on(DEVICE)
    freq = inv_freq(D).to(DEVICE)
    qkv = torch.zeros((rows, (NQ + 2 * NKV) * D), dtype=torch.bfloat16, device=DEVICE)
    q, out = (torch.zeros((rows, NQ * D), dtype=torch.bfloat16, device=DEVICE) for _ in range(2))
    positions, start_pos = torch.zeros(rows, **i32), torch.zeros(n, **i32)
    row_req = torch.arange(n, **i32).repeat_interleave(drafts + 1)
    starts = torch.arange(0, rows + 1, drafts + 1, **i32)
    logits, uniforms = torch.zeros((rows, VOCAB), device=DEVICE), torch.zeros(rows, device=DEVICE)
    drafted, temperatures = torch.zeros(n * drafts, **i32), torch.tensor([0.0, 0.7, 1.3], device=DEVICE)
    accepted, tokens = torch.zeros(n, **i32), torch.zeros(n, **i32)

    def step(c):
        ops.rope_kv_write_e4m3(qkv, NQ, NKV, D, freq, positions, row_req, c.table, PAGE, c.k, c.v, c.scale, q)
        ops.paged_attention_e4m3(q, NQ, NKV, D, c.k, c.v, c.scale, c.table, PAGE, starts, start_pos, n, drafts + 1, 200, None, 0.1, out)
        ops.verify_drafts(logits, None, drafted, starts, temperatures, uniforms, accepted, tokens)

    step(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).zero_()
    cache.scale.zero_()
    other = Cache([200] * n, NKV, D, PAGE).on(DEVICE)
    for turn in range(20):
        at = [turn * 3 + 40 * b for b in range(n)]
        start_pos.copy_(torch.tensor(at, dtype=torch.int32))
        positions.copy_(torch.tensor([p + j for p in at for j in range(drafts + 1)], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=gen))
        logits.copy_(3 * torch.randn(logits.shape, generator=gen))
        uniforms.copy_(torch.rand(rows, generator=gen))
        drafted.copy_(torch.randint(0, VOCAB, (n * drafts,), generator=gen))
        if turn % 2:
            drafted[0] = int(logits[0].argmax())
        graph.replay()
        got = [t.clone() for t in (q, out, accepted, tokens)]
        step(other)
        for a, b in zip(got, (q, out, accepted, tokens)):
            assert torch.equal(a, b), turn
        torch.cuda.synchronize()
    for a, b in ((cache.k, other.k), (cache.v, other.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(cache.scale, other.scale)
