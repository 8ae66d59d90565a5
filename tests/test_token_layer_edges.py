"""CPU: refusals of the token layers' example that need no GPU."""
import sys

import pytest

from tests.conftest import ROOT


def test_example_needs_a_step(monkeypatch):
    monkeypatch.syspath_prepend(str(ROOT / "examples"))
    import learned_stacks

    with pytest.raises(SystemExit, match="at least one step"):
        learned_stacks.main(steps=0)
    sys.modules.pop("learned_stacks")
