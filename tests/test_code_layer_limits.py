"""The layer example refuses what its caches do not hold, before it asks for a GPU."""

import sys

import pytest

from conftest import ROOT

sys.path.insert(0, str(ROOT / "examples"))


def test_more_steps_than_the_caches_hold():
    import code_layer

    with pytest.raises(ValueError, match="129 steps"):
        code_layer.main(2, code_layer.TOKENS + 1)
