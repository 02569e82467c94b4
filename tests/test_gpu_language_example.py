"""The example that runs the language-model operators together learns its rule and decodes it."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch  # noqa: F401  (before the library loads)

pytestmark = pytest.mark.gpu


def test_example_learns_and_decodes(gpu_ctx):
    path = Path(__file__).resolve().parent.parent / "examples" / "language_block.py"
    spec = importlib.util.spec_from_file_location("language_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, decoded, expected = example.main()
    # logits of standard deviation near 1 start near log(vocab) + 1/2; the rule leaves nothing to guess
    assert abs(losses[0] - math.log(example.VOCAB) - 0.5) < 0.5
    assert losses[-1] < 0.1 * losses[0]
    assert decoded == expected
