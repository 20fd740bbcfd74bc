"""Refusals of the speculative example, on the host."""

import pytest

from xpu_playground_b200.speculative import Server


def test_an_empty_prompt_is_refused():
    """It has no row whose logits say what comes first: another prompt's would be taken."""
    with pytest.raises(ValueError, match="at least one token"):
        Server.__new__(Server).generate([[1, 2], []], 4)
