"""examples/attention_layer.py: prompts, a resumed prompt and captured decode steps through the
projections, attention, the cache and the gate, against one prompt call without the cache."""
import os
import runpy
import sys

import pytest

from gpu_util import say

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_layer_agrees_with_itself(pkg, dev, monkeypatch, capsys):
    say("attention layer example")
    monkeypatch.setattr(sys, "argv", ["attention_layer.py", "--tokens", "40", "--check"])
    runpy.run_path(os.path.join(ROOT, "examples", "attention_layer.py"), run_name="__main__")
    out = capsys.readouterr().out
    assert "40 decoded each" in out and "largest difference" in out
