"""attention_tree over int8 caches with V scales of unusual sizes.

value = q * scale for any finite scale.  References and tolerance are those of
test_gpu_tree."""
import pytest
import torch
from test_gpu_tree import Batch

pytestmark = pytest.mark.gpu


def batch(shape, length, q_scale, seed=3):
    heads, nodes, n = shape
    return Batch("q8", *heads, lens=[length] * n, nodes=[nodes] * n, q_scale=q_scale, seed=seed)


def ordinary(b):
    """V scales as a quantiser makes them (test_gpu_tree spreads them by e^normal)."""
    b.cache.v_scale.copy_(torch.rand(b.cache.v_scale.shape, device="cuda") * 0.01 + 0.02)


@pytest.mark.parametrize("heads", [(4, 2, 100), (2, 2, 256)])
def test_values_whose_weighted_sum_passes_f32(gpu, heads):
    """A mean of values is no larger than they are, though their sum may be."""
    b = batch((heads, 2, 1), 300, 0.5)
    ordinary(b)
    for s in b.starts:  # int8 values of -1, 0 and 1, so that the values are finite
        b.cache.v[s + 5:s + 9].clamp_(-1, 1)
        b.cache.v_scale[s + 5:s + 9] = torch.tensor([2.0 ** 127, 2.0 ** 126, 3e38, 1e38], device="cuda")[:, None]
    b.check()
