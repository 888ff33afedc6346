"""A window of attention over 8-bit keys and values that 32 bits do not hold is as good as the widest that they hold (no GPU: the
kernel library is stood in for)."""
import pytest

from test_e4m3_refusals import attend, ops  # noqa: F401


@pytest.mark.parametrize("window,taken", [(None, 0), (1, 1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1),
                                          (2 ** 32 + 5, 2 ** 31 - 1), (10 ** 30, 2 ** 31 - 1)])
def test_the_window_that_the_library_gets(ops, window, taken):      # noqa: F811
    """(The call's 32-bit argument would take the low bits alone: a window of 5.)"""
    made = []
    ops.lib.__dict__["llmlab_paged_attention_e4m3"] = lambda *args: made.append(args) or 0
    ops.paged_attention_e4m3(**attend(window=window))
    assert [args[18] for args in made] == [taken]
