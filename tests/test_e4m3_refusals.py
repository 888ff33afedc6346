"""What the entry points of the 8-bit cache and of the check of drafted tokens refuse: all of it on the host,
before anything is launched (no GPU: the kernel libraries are stood in for)."""
import types

import pytest
import torch

from llm_inference_lab_amd.config.errors import UnsupportedSizeError
from llm_inference_lab_amd.kernels.hip_ops import HipOps

NQ, NKV, D, P, ROWS, PAGES, REQS = 4, 2, 32, 16, 5, 7, 3
F8, I32 = torch.float8_e4m3fn, torch.int32


class Calls:
    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        def call(*args):
            self.made.append(name)
            return 0
        return call


@pytest.fixture
def ops():
    x = object.__new__(HipOps)
    x.device = torch.device("cpu")
    x.calls_made, x._record = 0, None
    x.workspace = torch.zeros(1 << 16)
    x.num_cus = 256
    x.arrived = torch.zeros(64, dtype=I32)
    lib = Calls()
    x._mixer_lib = x._e4m3_attention_lib = lambda kind: lib
    x._stream = types.MethodType(lambda self: 0, x)
    x.lib = lib
    return x


def cache(**other):
    c = dict(k_cache=torch.zeros((PAGES, NKV, P, D), dtype=torch.uint8).view(F8),
             v_cache=torch.zeros((PAGES, NKV, D, P), dtype=torch.uint8).view(F8),
             kv_scale=torch.zeros((PAGES, NKV, 2, P), dtype=torch.uint8),
             block_table=torch.zeros((REQS, 4), dtype=I32), num_kv_heads=NKV, head_dim=D, page_size=P)
    c.update(other)
    return c


def write(**other):
    c = cache(qkv=torch.zeros((ROWS, (NQ + 2 * NKV) * D)), num_heads=NQ, inv_freq=torch.zeros(D // 2),
              positions=torch.zeros(ROWS, dtype=I32), row_req=torch.zeros(ROWS, dtype=I32), q_out=torch.zeros((ROWS, NQ * D)))
    c.update(other)
    return c


def read(**other):
    c = cache(positions=torch.zeros(ROWS, dtype=I32), row_req=torch.zeros(ROWS, dtype=I32), k_out=torch.zeros((ROWS, NKV * D)),
              v_out=torch.zeros((ROWS, NKV * D)))
    c.update(other)
    return c


def attend(**other):
    c = cache(q=torch.zeros((ROWS, NQ * D)), num_heads=NQ, q_start=torch.zeros(REQS + 1, dtype=I32),
              start_pos=torch.zeros(REQS, dtype=I32), n_reqs=REQS, max_q_len=2, max_ctx_len=40, window=None, scale=0.1,
              out=torch.zeros((ROWS, NQ * D)))
    c.update(other)
    return c


def verify(**other):
    c = dict(logits=torch.zeros((ROWS, 50)), draft_logits=torch.zeros((ROWS - REQS, 50)), drafts=torch.zeros(ROWS - REQS, dtype=I32),
             row_start=torch.zeros(REQS + 1, dtype=I32), temperatures=torch.zeros(REQS), uniforms=torch.zeros(ROWS),
             accepted=torch.zeros(REQS, dtype=I32), tokens=torch.zeros(REQS, dtype=I32))
    c.update(other)
    return c


def test_what_is_taken(ops):
    ops.rope_kv_write_e4m3(**write())
    ops.rope_kv_write_e4m3(**write(inv_freq=None, qkv=torch.zeros((ROWS, (NQ + 2 * NKV) * D), dtype=torch.bfloat16),
                                   q_out=torch.zeros((ROWS, NQ * D), dtype=torch.bfloat16)))
    ops.read_kv_e4m3(**read())
    ops.paged_attention_e4m3(**attend())
    ops.verify_drafts(**verify())
    ops.verify_drafts(**verify(draft_logits=None))
    assert len(ops.lib.made) == 6


CACHE = [
    (dict(k_cache=torch.zeros((PAGES, NKV, P, D), dtype=torch.uint8)), TypeError),
    (dict(k_cache=torch.zeros((PAGES, NKV, D, P), dtype=torch.uint8).view(F8)), ValueError),
    (dict(k_cache=torch.zeros((PAGES, NKV, P, 2 * D), dtype=torch.uint8).view(F8)[..., :D]), ValueError),
    (dict(v_cache=torch.zeros((PAGES + 1, NKV, D, P), dtype=torch.uint8).view(F8)), ValueError),
    (dict(v_cache=torch.zeros(PAGES * NKV * D * P + 1, dtype=torch.uint8)[1:].view(F8).view(PAGES, NKV, D, P)), ValueError),
    (dict(kv_scale=torch.zeros((PAGES, NKV, P, 2), dtype=torch.uint8)), ValueError),
    (dict(kv_scale=torch.zeros((PAGES, NKV, 2, P), dtype=torch.int8)), TypeError),
    (dict(block_table=torch.zeros((REQS, 4), dtype=torch.int64)), TypeError),
    (dict(block_table=torch.zeros((REQS, 8), dtype=I32)[:, ::2]), ValueError),
    (dict(page_size=8), UnsupportedSizeError),
    (dict(page_size=24), UnsupportedSizeError),
    (dict(head_dim=24), (UnsupportedSizeError, ValueError)),
    (dict(head_dim=272), (UnsupportedSizeError, ValueError)),
    (dict(block_table=torch.zeros((REQS, 4), dtype=I32, device="meta")), ValueError),
]


@pytest.mark.parametrize("other,error", CACHE)
@pytest.mark.parametrize("name", ["write", "read", "attend"])
def test_caches_that_do_not_fit(ops, name, other, error):
    call, args = {"write": (ops.rope_kv_write_e4m3, write), "read": (ops.read_kv_e4m3, read),
                  "attend": (ops.paged_attention_e4m3, attend)}[name]
    with pytest.raises(error):
        call(**args(**other))
    assert not ops.lib.made


@pytest.mark.parametrize("other,error", [
    (dict(qkv=torch.zeros((ROWS, (NQ + 2 * NKV) * D), dtype=torch.float16)), TypeError),
    (dict(qkv=torch.zeros((ROWS, (NQ + NKV) * D))), ValueError),
    (dict(qkv=torch.zeros(((NQ + 2 * NKV) * D, ROWS)).t()), ValueError),
    (dict(q_out=torch.zeros((ROWS, NQ * D), dtype=torch.bfloat16)), TypeError),
    (dict(q_out=torch.zeros((ROWS - 1, NQ * D))), ValueError),
    (dict(positions=torch.zeros(ROWS - 1, dtype=I32)), ValueError),
    (dict(row_req=torch.zeros(ROWS)), TypeError),
    (dict(inv_freq=torch.zeros(D)), ValueError),
    (dict(inv_freq=torch.zeros(D // 2, dtype=torch.float64)), TypeError),
])
def test_writes(ops, other, error):
    with pytest.raises(error):
        ops.rope_kv_write_e4m3(**write(**other))
    assert not ops.lib.made


@pytest.mark.parametrize("other,error", [
    (dict(k_out=torch.zeros((ROWS, NKV * D), dtype=torch.float16)), TypeError),
    (dict(v_out=torch.zeros((ROWS, NKV * D), dtype=torch.bfloat16)), TypeError),
    (dict(v_out=torch.zeros((ROWS, D))), ValueError),
    (dict(k_out=torch.zeros((ROWS, 2 * NKV * D))[:, ::2]), ValueError),
    (dict(positions=torch.zeros(ROWS - 1, dtype=I32)), ValueError),
])
def test_reads(ops, other, error):
    with pytest.raises(error):
        ops.read_kv_e4m3(**read(**other))
    assert not ops.lib.made


@pytest.mark.parametrize("other,error", [
    (dict(q=torch.zeros((ROWS, NQ * D), dtype=torch.float16)), TypeError),
    (dict(q=torch.zeros((ROWS, NQ * D - 1))), ValueError),
    (dict(q=torch.zeros((ROWS, NQ * D + 1))), ValueError),
    (dict(out=torch.zeros((ROWS, NQ * D), dtype=torch.bfloat16)), TypeError),
    (dict(out=torch.zeros((ROWS + 1, NQ * D))), ValueError),
    (dict(num_heads=3, q=torch.zeros((ROWS, 3 * D)), out=torch.zeros((ROWS, 3 * D))), UnsupportedSizeError),
    (dict(n_reqs=REQS + 1), ValueError),
    (dict(n_reqs=-1), ValueError),
    (dict(max_ctx_len=4 * P + 1), ValueError),
    (dict(q_start=torch.zeros(REQS, dtype=I32)), ValueError),
    (dict(start_pos=torch.zeros(REQS, dtype=torch.int64)), TypeError),
    (dict(window=0), ValueError),
    (dict(window=-3), ValueError),
])
def test_attention(ops, other, error):
    with pytest.raises(error):
        ops.paged_attention_e4m3(**attend(**other))
    assert not ops.lib.made


@pytest.mark.parametrize("other,error", [
    (dict(logits=torch.zeros((ROWS, 50), dtype=torch.bfloat16)), TypeError),
    (dict(logits=torch.zeros((50, ROWS)).t()), ValueError),
    (dict(logits=torch.zeros((ROWS, 0))), ValueError),
    (dict(logits=torch.zeros((REQS - 1, 50)), draft_logits=None), ValueError),
    (dict(draft_logits=torch.zeros((ROWS, 50))), ValueError),
    (dict(draft_logits=torch.zeros((ROWS - REQS, 49))), ValueError),
    (dict(drafts=torch.zeros(ROWS - REQS - 1, dtype=I32)), ValueError),
    (dict(drafts=torch.zeros(ROWS - REQS, dtype=torch.int64)), TypeError),
    (dict(row_start=torch.zeros(0, dtype=I32)), ValueError),
    (dict(temperatures=torch.zeros(REQS - 1)), ValueError),
    (dict(uniforms=torch.zeros(ROWS - 1)), ValueError),
    (dict(uniforms=torch.zeros(ROWS, dtype=torch.float64)), TypeError),
    (dict(accepted=torch.zeros(REQS - 1, dtype=I32)), ValueError),
    (dict(tokens=torch.zeros(REQS, dtype=torch.int64)), TypeError),
])
def test_verification(ops, other, error):
    with pytest.raises(error):
        ops.verify_drafts(**verify(**other))
    assert not ops.lib.made
