"""Calls of the serving operators that would leave outputs unwritten, without a GPU."""

import pytest

from tests.test_serving_host import INVALID, PROMPT
from xpu_playground_b200 import _lib


def test_a_plan_without_tiles_is_refused_where_there_are_tokens():
    assert _lib.load().xpu_prompt_attention(*(PROMPT | {"blocks": 0}).values(), None) == INVALID
    assert "no tiles" in _lib.last_error()
    assert _lib.load().xpu_prompt_attention(*(PROMPT | {"blocks": 0, "tokens": 0}).values(), None) == 0
