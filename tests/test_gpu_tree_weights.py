"""attention_tree over an int8 cache: weights far below the largest still count.

A place whose score lies far above the rest takes nearly all the weight.  What the
others add is a small part of the output, but there are many of them.

Tolerance, for each (node, head) row.  A place's probability p_j has the relative
error e_j of its score, (8 + sqrt(hd)) * 2^-24 * max(S_j, 1) with S_j = sum |q_d k_d| /
sqrt(hd) (see test_gpu_tree); the softmax's division takes the common part out, so the
output's error is at most sum_j p_j e_j |v_j - out|.  Products and sums of f32 add
8 * 2^-24 * sum_j p_j |v_j|.  The first sum takes little from the large score, since out
is next to that place's value: the bound does not grow with it."""
import math

import pytest
import torch

from prana_b200 import kernels as K

pytestmark = pytest.mark.gpu


def run(n_seq, length, n_heads, n_kv, hd, nodes, tops, seed=0, empty_dims=0):
    """Sequences whose places tops = {place: score above the mean} stand out; the worst row's error over its bound."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = length + nodes
    cache = K.KvRows.alloc(n_seq * rows, n_kv, hd, quantized=True)
    one = torch.ones(hd, device="cuda") / math.sqrt(hd)
    where = torch.arange(n_seq * rows, dtype=torch.int32, device="cuda").view(n_seq, rows)
    for b in range(n_seq):
        k, v = (torch.randn(rows, n_kv, hd, generator=g, device="cuda") for _ in range(2))
        k -= (k @ one)[..., None] * one  # across q's common direction
        k += torch.randn(rows, n_kv, 1, generator=g, device="cuda") * 0.05 * one
        for place, top in tops.items():
            k[place] = one * top
            v[place, :, :empty_dims] = 0.0
        K.kv_rows_write(cache, where[b], k, v)
    q = torch.randn(n_seq * nodes, n_heads, hd, generator=g, device="cuda") * 0.3
    q += (math.sqrt(hd) - q @ one)[..., None] * one  # score of k = one * t: t
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = K.attention_tree(q.view(n_seq * nodes, -1), cache, i32([b * rows for b in range(n_seq)]), i32([length] * n_seq),
                           i32([b * nodes for b in range(n_seq + 1)]), nodes, n_heads)
    K.synchronize()
    out = out.view(n_seq, nodes, n_heads, hd).double()
    worst = 0.0
    for b in sorted({0, n_seq // 2, n_seq - 1}):
        k, v = (x.double() for x in K.kv_rows_read(cache, where[b]))
        for i in range(nodes):
            at = length + i + 1
            for h in range(n_heads):
                c, x = h // (n_heads // n_kv), q[b * nodes + i, h].double()
                kk, vv = k[:at, c], v[:at, c]
                p = torch.softmax(kk @ x / math.sqrt(hd), 0)
                ref = p @ vv
                e = (8 + math.sqrt(hd)) * 2.0 ** -24 * (kk.abs() @ x.abs() / math.sqrt(hd)).clamp(min=1.0)
                bound = (p * e * (vv - ref).norm(dim=1)).sum() + 8 * 2.0 ** -24 * (p * vv.norm(dim=1)).sum()
                worst = max(worst, float((out[b, i, h] - ref).norm() / bound))
    return worst


# 8, 16, 32 and 64 columns of a kv head; sequences enough that a unit's tiles lie in one share
WIDTHS = [(32, 8, 128, 1), (32, 8, 128, 4), (32, 8, 128, 8), (32, 8, 128, 16)]


@pytest.mark.parametrize("top", [0.0, 12.0, 16.0, 18.0, 22.0])
@pytest.mark.parametrize("heads", WIDTHS)
def test_one_score_above_the_rest(gpu, top, heads):
    assert run(20, 16384, *heads, {5: top}) <= 1.0


@pytest.mark.parametrize("top", [12.0, 18.0])
@pytest.mark.parametrize("heads", [WIDTHS[0], WIDTHS[2]])
def test_one_score_above_a_long_context(gpu, top, heads):
    assert run(19, 32000, *heads, {31000: top}) <= 1.0


@pytest.mark.parametrize("heads", WIDTHS)
@pytest.mark.parametrize("places", [(5, 700), (2000, 2100, 2300, 9000), tuple(range(300, 1500))])
def test_several_scores_above_the_rest(gpu, heads, places):
    assert run(20, 16384, *heads, {p: 17.0 for p in places}) <= 1.0


@pytest.mark.parametrize("heads", WIDTHS)
def test_levels_that_fall(gpu, heads):
    """Stretches of 1000 places, each 4 below the one before."""
    assert run(20, 8000, *heads, {p: 16.0 - 4.0 * (p // 1000) for p in range(5000)}) <= 1.0


@pytest.mark.parametrize("n_seq", [1, 20])
def test_dims_that_the_large_score_leaves_to_the_rest(gpu, n_seq):
    assert run(n_seq, 16384, 32, 8, 128, 1, {5: 14.0}, empty_dims=64) <= 1.0
