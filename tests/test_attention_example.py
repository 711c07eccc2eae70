"""The example's options: what it cannot run with is said before anything runs."""
import importlib.util
import os

import pytest

spec = importlib.util.spec_from_file_location(
    "attend_example", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vectorlink-gpu_amd", "attend.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def test_every_option_is_a_number_of_one_or_more(capsys):
    options = example.parse([])
    assert all(options[long_[2:]] == default for (_, long_, default, _) in example.INT_OPTIONS)
    for short, long_, _, _ in example.INT_OPTIONS:
        assert example.parse([short, "7"])[long_[2:]] == 7
        for bad in ("0", "-3", "some"):
            with pytest.raises(SystemExit):
                example.parse([long_, bad])
    assert "at least 1" in capsys.readouterr().err
