"""examples/tree_decode.py: trees of drafted tokens give the tokens of one at a time."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "tree_decode.py"
    spec = importlib.util.spec_from_file_location("tree_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("branches", [(1, 1, 1), (3, 2, 1), (2, 2, 2, 2)])
def test_same_tokens_in_fewer_steps(example, quantized, branches):
    model = example.Transformer()
    prompt = [(7 * i * i + 3) % 512 for i in range(100)]
    plain, passes = example.generate(model, prompt, 3, 40, quantized, ())
    assert passes == 39
    text, steps = example.generate(model, prompt, 3, 40, quantized, branches)
    assert text == plain
    assert steps < passes
    assert len({tuple(t) for t in text}) == 3
