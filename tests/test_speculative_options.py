"""The speculative example's options, on the host."""

import pytest

from xpu_playground_b200.speculative import main


@pytest.mark.parametrize("option", [["--top-k", "5"], ["--top-p", "0.9"], ["--min-p", "0.1"]])
def test_settings_of_drawing_need_a_temperature(option, capsys):
    with pytest.raises(SystemExit):
        main(option)
    assert "need --temperature" in capsys.readouterr().err
