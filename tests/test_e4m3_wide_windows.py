"""A window of attention over 8-bit keys and values, or a bound on its portions and contexts, that 32 bits do not hold is as good as the
widest that they hold (no GPU: the kernel library is stood in for)."""
import pytest
import torch

from test_e4m3_refusals import attend, ops  # noqa: F401


@pytest.mark.parametrize("window,taken", [(None, 0), (1, 1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1),
                                          (2 ** 32 + 5, 2 ** 31 - 1), (10 ** 30, 2 ** 31 - 1)])
def test_the_window_that_the_library_gets(ops, window, taken):      # noqa: F811
    """(The call's 32-bit argument would take the low bits alone: a window of 5.)"""
    made = []
    ops.lib.__dict__["llmlab_paged_attention_e4m3"] = lambda *args: made.append(args) or 0
    ops.paged_attention_e4m3(**attend(window=window))
    assert [args[18] for args in made] == [taken]


@pytest.mark.parametrize("longest,taken", [(2, 2), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32, 2 ** 31 - 1)])
def test_the_longest_portion_that_the_library_gets(ops, longest, taken):      # noqa: F811
    """(The low bits of 2^31 are a negative number, of 2^32 none: nothing would be attended to.)"""
    made = []
    ops.lib.__dict__["llmlab_paged_attention_e4m3"] = lambda *args: made.append(args) or 0
    ops.paged_attention_e4m3(**attend(max_q_len=longest))
    assert [args[16] for args in made] == [taken]


def test_the_longest_context_that_the_library_gets(ops):      # noqa: F811
    """A table that has room for more than 2^31 keys."""
    made = []
    ops.lib.__dict__["llmlab_paged_attention_e4m3"] = lambda *args: made.append(args) or 0
    wide = torch.zeros((3, 1), dtype=torch.int32).expand(3, 2 ** 28)      # (a stride of 0: no memory; 2^32 keys of pages of 16)
    with pytest.raises(ValueError):
        ops.paged_attention_e4m3(**attend(block_table=wide, max_ctx_len=2 ** 31 + 5))
    call = ops.prepare_attention_e4m3(*(attend()[n] for n in (
        "q", "num_heads", "num_kv_heads", "head_dim", "k_cache", "v_cache", "kv_scale", "block_table", "page_size", "q_start",
        "start_pos", "window", "scale", "out")))
    call.most_context = 2 ** 32
    call.launch(3, 2, 2 ** 31 + 5)
    assert [args[17] for args in made] == [2 ** 31 - 1]
