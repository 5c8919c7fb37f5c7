"""attention_tree over int8 caches whose V scales are zero, tiny, huge or negative.

value = q * scale for any finite scale, so such a place takes part like another:
its weight counts in the softmax's sum whatever its scale.  References and
tolerance are those of test_gpu_tree."""
import numpy as np
import pytest
import torch
from test_gpu_tree import Batch

pytestmark = pytest.mark.gpu

# (heads, nodes, sequences): 8, 16, 32 and 64 columns share a kv head, and a head size without tensor cores
SHAPES = [((8, 2, 128), 2, 1), ((8, 2, 64), 4, 2), ((8, 2, 128), 8, 2), ((8, 2, 128), 15, 9), ((4, 2, 100), 2, 1)]


def batch(shape, length, q_scale, seed=3):
    heads, nodes, n = shape
    return Batch("q8", *heads, lens=[length] * n, nodes=[nodes] * n, q_scale=q_scale, seed=seed)


def ordinary(b):
    """V scales as a quantiser makes them (test_gpu_tree spreads them by e^normal)."""
    b.cache.v_scale.copy_(torch.rand(b.cache.v_scale.shape, device="cuda") * 0.01 + 0.02)


@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-40])
@pytest.mark.parametrize("q_scale", [0.3, 0.7, 2.0])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("length,rows", [(512, (0, 128)), (390, (384, 390)), (392, (384, 392)), (4000, (0, 2304)), (4000, (128, 4000))])
def test_context_rows_without_a_value(gpu, shape, length, rows, q_scale, scale):
    b = batch(shape, length, q_scale)
    ordinary(b)
    for s in b.starts:
        b.cache.v_scale[s + rows[0]:s + rows[1]] = scale
    b.check()


@pytest.mark.parametrize("scale", [0.0, 1e-38])
@pytest.mark.parametrize("q_scale", [0.3, 0.7, 2.0])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("length", [0, 128, 300])
def test_drafted_rows_without_a_value(gpu, shape, length, q_scale, scale):
    b = batch(shape, length, q_scale)
    ordinary(b)
    for s in b.starts:
        b.cache.v_scale[s + length:s + length + shape[1]] = scale
    b.check()


@pytest.mark.parametrize("shape", SHAPES)
def test_no_value_at_all(gpu, shape):
    b = batch(shape, 700, 0.7)
    b.cache.v_scale.zero_()
    out = b.run()
    assert int(out.count_nonzero()) == 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e-18, 1e18, 1e30])
def test_a_whole_cache_of_one_size(gpu, shape, scale):
    b = batch(shape, 700, 1.0)
    ordinary(b)
    b.cache.v_scale.mul_(scale)
    b.check()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("first,second", [(1e25, 1e-25), (1e-25, 1e25), (1e30, 1.0), (1.0, 1e-20), (0.0, 1e36)])
def test_two_sizes_side_by_side(gpu, shape, first, second):
    b = batch(shape, 900, 0.5)
    ordinary(b)
    for s in b.starts:
        b.cache.v_scale[s:s + 450] *= first
        b.cache.v_scale[s + 450:s + 900 + shape[1]] *= second
    b.check()


@pytest.mark.parametrize("shape", SHAPES)
def test_the_largest_scales(gpu, shape):
    b = batch(shape, 300, 0.5)
    ordinary(b)
    for s in b.starts:  # int8 values of -1, 0 and 1, so that the values are finite
        b.cache.v[s + 5:s + 9].clamp_(-1, 1)
        b.cache.v_scale[s + 5:s + 9] = torch.tensor([2.0 ** 127, 2.0 ** 126, 3e38, 1e38], device="cuda")[:, None]
    b.check()


@pytest.mark.parametrize("shape", SHAPES)
def test_a_place_without_a_value_takes_nearly_all_the_weight(gpu, shape):
    """What is left of the others' weight is their values' share of it."""
    b = batch(shape, 600, 0.1)
    ordinary(b)
    hd = b.shape[2]
    for s in b.starts:
        b.cache.k[s + 200] = 127
        b.cache.k_scale[s + 200] = 1.0 / 127
        b.cache.v_scale[s + 200] = 0.0
    b.q += 12.0 / np.sqrt(hd)
    b.check()


@pytest.mark.parametrize("columns,n", [(2, 1), (8, 2), (15, 9)])
def test_a_nan_score_of_a_place_without_a_value_is_not_hidden(gpu, columns, n):
    b = batch(((8, 2, 128), columns, n), 300, 1.0)
    b.cache.v_scale[b.starts[0] + 130] = 0.0
    b.cache.k_scale[b.starts[0] + 130] = float("nan")
    out = b.run()
    assert torch.isnan(out[:columns]).all() and torch.isfinite(out[columns:]).all()


@pytest.mark.parametrize("heads", [(4, 2, 100), (2, 2, 256)])
def test_values_whose_weighted_sum_passes_f32(gpu, heads):
    """A mean of values is no larger than they are, though their sum may be."""
    b = batch((heads, 2, 1), 300, 0.5)
    ordinary(b)
    for s in b.starts:  # int8 values of -1, 0 and 1, so that the values are finite
        b.cache.v[s + 5:s + 9].clamp_(-1, 1)
        b.cache.v_scale[s + 5:s + 9] = torch.tensor([2.0 ** 127, 2.0 ** 126, 3e38, 1e38], device="cuda")[:, None]
    b.check()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("q_scale", [0.5, 3.0])
@pytest.mark.parametrize("length", [5, 700, 4000])
def test_negative_scales(gpu, shape, q_scale, length):
    b = batch(shape, length, q_scale)
    for x in (b.cache.k_scale, b.cache.v_scale):
        x[1::2] *= -1.0
    for s in b.starts:
        b.cache.v_scale[s + 2] = -0.0
    b.check()
