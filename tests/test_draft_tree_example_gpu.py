"""The draft-tree example runs, and its attention agrees with plain torch from
the cache read back: as a whole within 2^-8, of which rounding the output to bf16
is up to 2^-9 and rounding probabilities and values to f16 up to 2^-10 of terms
that add up at random."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["block", "mxfp8", "nvfp4"])
def test_draft_tree(name):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "draft_tree.py")
    spec = importlib.util.spec_from_file_location("draft_tree", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, error, out = m.main(name)
    assert losses[-1] < losses[0]
    assert error < 2.0 ** -8
    assert bool(out.isfinite().all())
