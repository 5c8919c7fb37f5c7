"""Attention over trees of drafted tokens against a 64-bit restatement.

Tolerance.  Each score is rounded a few times in f32, and its products carry
about 22 bits or more, so its error is near 2^-24 times the sum of |q_d k_d| /
sqrt(hd) (call the largest S) times a small count; a sequential f32 sum adds
about sqrt(hd) more of them.  A score's error is a relative error of its
probability, and the output is a weighted mean.  So the 2-norm error relative
to the output's is held to (8 + sqrt(hd)) * 2^-24 * max(S, 1)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from prana_b200 import _ffi
from prana_b200 import kernels as K
from prana_b200._ffi import PranaError

pytestmark = pytest.mark.gpu


def random_tree(rng, n):
    return [-1 if i == 0 else int(rng.integers(max(0, i - 6), i)) for i in range(n)]


class Batch:
    """A ragged batch in one cache: sequence b has lens[b] context rows and nodes[b] drafted tokens."""

    def __init__(self, kind, n_heads, n_kv, hd, lens, nodes, seed=0, masks="tree", gap=3, layout="rows", q_scale=1.5):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.shape = (n_heads, n_kv, hd)
        self.lens, self.nodes, self.max_nodes = list(lens), list(nodes), max(max(nodes), 1)
        room = [a + b + gap for a, b in zip(lens, nodes)]
        self.starts = [gap + sum(room[:b]) for b in range(len(room))]
        positions = gap + sum(room)
        k, v = (torch.randn(positions, n_kv, hd, generator=g, device="cuda") + 0.3 for _ in range(2))
        if kind == "q8":
            ks, vs = k.abs().amax(-1) / 127, v.abs().amax(-1) / 127 * torch.exp(torch.randn(positions, n_kv, generator=g, device="cuda"))
            k, v = torch.round(k / ks[..., None]).to(torch.int8), torch.randint(-127, 128, k.shape, generator=g, device="cuda", dtype=torch.int8)
            if layout == "heads":
                k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
                ks, vs = ks.t().contiguous().t(), vs.t().contiguous().t()
        else:
            k, v, ks, vs = k.half(), v.half(), None, None
            if layout == "heads":
                k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
        if layout == "slice":
            def inside(x):
                wide = torch.zeros(positions, n_kv, hd + 3, dtype=x.dtype, device="cuda")
                wide[:, :, 1:1 + hd] = x
                return wide[:, :, 1:1 + hd]
            k, v = inside(k), inside(v)
        self.cache = K.KvRows(k, v, ks, vs)
        self.q = torch.randn(sum(nodes), n_heads * hd, generator=g, device="cuda") * q_scale
        self.offsets = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.masks = None
        if masks == "tree":
            self.masks = [m for n in nodes for m in K.tree_masks(random_tree(rng, n))] if sum(nodes) else []
        elif masks == "random":  # any bits, rows that see nothing of the draft among them, bits past the last node too
            self.masks = [int(x) for x in rng.integers(-2 ** 63, 2 ** 63, sum(nodes)) & np.where(rng.random(sum(nodes)) < 0.3, 0, -1)]

    def run(self, **more):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        masks = None if self.masks is None else torch.tensor(self.masks, dtype=torch.int64, device="cuda")
        return K.attention_tree(self.q, self.cache, i32(self.starts), i32(self.lens), i32(self.offsets.tolist()),
                                self.max_nodes, self.shape[0], masks, **more)

    def see(self, b):
        n, mask = self.nodes[b], np.zeros((self.nodes[b], self.lens[b] + self.nodes[b]), bool)
        mask[:, : self.lens[b]] = True
        for i in range(n):
            m = (2 << i) - 1 if self.masks is None else self.masks[self.offsets[b] + i]
            mask[i, self.lens[b]:] = [bool(m >> j & 1) for j in range(n)]
        return mask

    def reference(self):
        """(out, S) in float64: each row of a place it does not see is left out, not multiplied by zero."""
        nh, n_kv, hd = self.shape
        out, biggest = np.zeros((sum(self.nodes), nh, hd)), 0.0
        q = self.q.cpu().numpy().astype(np.float64).reshape(-1, nh, hd)
        for b, n in enumerate(self.nodes):
            rows = slice(self.starts[b], self.starts[b] + self.lens[b] + n)
            k, v = (x[rows].cpu().numpy().astype(np.float64) for x in (self.cache.k, self.cache.v))
            if self.cache.quantized:
                k = k * self.cache.k_scale[rows].cpu().numpy().astype(np.float64)[..., None]
                v = v * self.cache.v_scale[rows].cpu().numpy().astype(np.float64)[..., None]
            see = self.see(b)
            for i in range(n):
                at = np.flatnonzero(see[i])
                if not len(at):
                    continue
                for h in range(nh):
                    c, x = h // (nh // n_kv), q[self.offsets[b] + i, h]
                    s = k[at, c] @ x / math.sqrt(hd)
                    with np.errstate(invalid="ignore"):
                        biggest = max(biggest, float(np.nanmax(np.abs(k[at, c]) @ np.abs(x))) / math.sqrt(hd))
                    p = np.exp(s - s.max())
                    out[self.offsets[b] + i, h] = p @ v[at, c] / p.sum()
        return out.reshape(sum(self.nodes), nh * hd), biggest

    def check(self, got=None):
        got = (self.run() if got is None else got).cpu().numpy().astype(np.float64)
        K.synchronize()
        ref, biggest = self.reference()
        tol = (8 + math.sqrt(self.shape[2])) * 2.0 ** -24 * max(biggest, 1.0)
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        fine = ~np.isnan(ref)
        assert np.linalg.norm(got[fine] - ref[fine]) <= tol * np.linalg.norm(ref[fine])
        # and every (node, head) row by itself, with room for one row's luck
        width = self.shape[2]
        d, r = (np.linalg.norm(np.where(fine, x, 0).reshape(-1, width), axis=1) for x in (got - ref, ref))
        assert np.all(d <= 8 * tol * np.maximum(r, np.sqrt(np.mean(r ** 2)) if len(r) else 0))


HEADS = [(32, 8, 128), (14, 2, 64), (6, 6, 48), (4, 1, 128), (9, 3, 96), (8, 1, 32), (5, 1, 16), (2, 2, 256), (6, 2, 100), (71, 1, 64)]


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("heads", HEADS)
def test_decode_ragged(gpu, kind, heads):
    Batch(kind, *heads, lens=[0, 1, 127, 128, 129, 700], nodes=[1] * 6, masks=None).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("masks", ["tree", "random", None])
def test_trees_ragged(gpu, kind, heads, masks):
    Batch(kind, *heads, lens=[0, 5, 126, 250, 300], nodes=[7, 0, 3, 12, 1], masks=masks, seed=2).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (6, 6, 48)])
@pytest.mark.parametrize("length,nodes", [(0, 64), (1, 64), (64, 64), (65, 63), (127, 2), (128, 33), (1000, 17)])
def test_largest_trees_and_tile_edges(gpu, kind, heads, length, nodes):
    Batch(kind, *heads, lens=[length, length + 3], nodes=[nodes, 1], masks="tree", seed=nodes).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("nodes", [1, 2, 3, 4, 5, 8, 9, 16, 40])
def test_every_width(gpu, kind, nodes):
    Batch(kind, 16, 4, 128, lens=[333, 4000], nodes=[nodes, nodes], seed=nodes).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("layout", ["heads", "slice"])
@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (6, 6, 48)])
def test_layouts(gpu, kind, layout, heads):
    Batch(kind, *heads, lens=[100, 257], nodes=[6, 9], layout=layout).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("nodes", [1, 12])
def test_long_context(gpu, kind, nodes):
    Batch(kind, 8, 2, 128, lens=[33333], nodes=[nodes]).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_many_short_sequences(gpu, kind):
    rng = np.random.default_rng(0)
    n = 700
    Batch(kind, 4, 2, 64, lens=rng.integers(0, 150, n).tolist(), nodes=rng.integers(0, 4, n).tolist()).check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("nodes", [1, 9, 40])
def test_sharp_and_flat_scores(gpu, kind, nodes):
    Batch(kind, 8, 2, 128, lens=[900, 900], nodes=[nodes, nodes], q_scale=30.0).check()
    b = Batch(kind, 8, 2, 128, lens=[900], nodes=[nodes], q_scale=1.0)
    b.q.zero_()  # every place alike
    b.check()
    b.q.fill_(1e-30)
    b.check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("nodes", [1, 12])
def test_one_place_takes_nearly_all_the_weight(gpu, kind, nodes):
    """A first row with a far larger score and a tiny value: what is left of the others still counts."""
    b = Batch(kind, 4, 1, 128, lens=[3000], nodes=[nodes], masks=None)
    first = b.starts[0]
    if kind == "q8":
        b.cache.v_scale[first] = 1e-9
        b.cache.k[first] = 127
        b.cache.k_scale[first] = 1.0 / 127
    else:
        b.cache.v[first] = 1e-7
        b.cache.k[first] = 1.0
    b.q[:] = b.q * 0.1 + 16.0 / math.sqrt(128)
    b.cache.k[first + 1: first + 3000] -= b.cache.k[first + 1: first + 3000] // 2
    b.check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("nodes", [1, 5, 40])
def test_rows_not_in_use_may_hold_anything(gpu, kind, nodes):
    b = Batch(kind, 8, 2, 64, lens=[0, 100, 128, 200], nodes=[nodes] * 4)
    used = torch.zeros(b.cache.k.shape[0], dtype=torch.bool, device="cuda")
    for s, n in zip(b.starts, b.lens):
        used[s:s + n + nodes] = True
    if kind == "q8":
        for x, bad in ((b.cache.k_scale, math.nan), (b.cache.v_scale, math.inf)):
            x[~used] = bad
        b.cache.k[~used], b.cache.v[~used] = -128, 127
    else:
        b.cache.k[~used], b.cache.v[~used] = math.nan, math.inf
    b.check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 4, 128), (6, 2, 100)])
def test_what_a_node_does_not_see_has_no_effect(gpu, kind, what, heads):
    """A drafted row of NaN reaches the nodes that see it, and no others."""
    b = Batch(kind, *heads, lens=[130, 20], nodes=[16, 16], masks="tree", seed=4)
    clean = b.run().clone()
    for seq, node in ((0, 3), (1, 15)):
        row = b.starts[seq] + b.lens[seq] + node
        if kind == "q8":
            getattr(b.cache, what + "_scale")[row] = math.nan
        else:
            getattr(b.cache, what)[row] = math.nan
    got = b.run()
    K.synchronize()
    for seq, node in ((0, 3), (1, 15)):
        hit = torch.tensor(b.see(seq)[:, b.lens[seq] + node], device="cuda")
        rows = slice(b.offsets[seq], b.offsets[seq + 1])
        assert torch.isnan(got[rows][hit]).all() and int(hit.sum()) >= 1
        assert torch.equal(got[rows][~hit], clean[rows][~hit]) and int((~hit).sum()) >= 1


@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_nodes_that_see_nothing_get_zeros(gpu, kind):
    b = Batch(kind, 8, 2, 128, lens=[0, 40], nodes=[4, 4], masks="tree")
    b.masks = [1, 0, 0b100, 0, 0, 1, 0, 0b1000]
    out = b.run()
    b.check(out)
    assert int(out[1].count_nonzero()) == 0 and int(out[3].count_nonzero()) == 0
    assert int(out[4].count_nonzero()) > 0  # its context remains


@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_a_nan_in_the_context_or_the_query_is_not_hidden(gpu, kind):
    b = Batch(kind, 8, 2, 64, lens=[300, 300], nodes=[3, 3], masks=None)
    if kind == "q8":
        b.cache.k_scale[b.starts[0] + 7] = math.nan
    else:
        b.cache.k[b.starts[0] + 7] = math.nan
    b.q[4, 64:128] = math.nan  # one head of one node
    out = b.run()
    K.synchronize()
    assert torch.isnan(out[:3]).all()
    want = torch.zeros(3, 8 * 64, dtype=torch.bool, device="cuda")
    want[1, 64:128] = True
    assert torch.equal(torch.isnan(out[3:]), want)


@pytest.mark.parametrize("hd,n_heads,n_kv", [(64, 14, 2), (128, 32, 8), (48, 6, 6)])
def test_a_chain_is_attention_verify(gpu, hd, n_heads, n_kv):
    """masks None over one f16 sequence: the values of attention_verify and attention_decode."""
    pos0, n = 301, 5
    b = Batch("f16", n_heads, n_kv, hd, lens=[pos0], nodes=[n], masks=None, gap=0)
    kc, vc = (x.reshape(-1, n_kv * hd) for x in (b.cache.k, b.cache.v))
    ref = K.attention_verify(b.q, kc, vc, pos0, n, n_heads, n_kv, hd)
    one = K.attention_decode(b.q[0].contiguous(), kc, vc, pos0, n_heads, n_kv, hd)
    got = b.run()
    K.synchronize()
    assert float((got - ref).norm() / ref.norm()) < 2e-5  # the kernels' own tolerance, twice
    assert float((got[0] - one).norm() / one.norm()) < 2e-5


@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_the_same_bits_every_time_and_on_any_stream(gpu, kind):
    b = Batch(kind, 32, 8, 128, lens=[2000, 3, 700], nodes=[9, 9, 9])
    other = Batch(kind, 32, 8, 128, lens=[90, 1500, 7], nodes=[16, 2, 30], seed=9)
    first, second = b.run().clone(), other.run().clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):  # two batches at once, each on its own stream
        for s, x in zip(streams, (b, other)):
            with torch.cuda.stream(s):
                outs.append(x.run())
    torch.cuda.synchronize()
    assert all(torch.equal(o, (first, second)[i % 2]) for i, o in enumerate(outs))


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("heads,lens,nodes", [((32, 8, 128), [9000, 1, 4000, 130, 7000] * 3, [1] * 15), ((32, 8, 128), [3000, 129, 600] * 4, [20, 1, 60] * 4),
                                              ((14, 2, 64), [40, 3, 300, 90] * 50, [2, 5, 1, 9] * 50)])
def test_many_runs_give_one_answer(gpu, kind, heads, lens, nodes):
    """Long and short units side by side in every share, over and over: no wait runs out, no tile is taken for another."""
    b = Batch(kind, *heads, lens=lens, nodes=nodes)
    want = b.run().clone()
    for _ in range(60):
        assert torch.equal(b.run(), want)
    K.synchronize()
    b.check(want)


@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_captured_into_a_graph(gpu, kind):
    b = Batch(kind, 8, 2, 128, lens=[500, 40], nodes=[5, 5])
    want = b.run().clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (i32(b.starts), i32(b.lens), i32(b.offsets.tolist()), 5, 8, torch.tensor(b.masks, device="cuda"))
    out = torch.empty_like(want)
    K.attention_tree(b.q, b.cache, *args, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.attention_tree(b.q, b.cache, *args, out=out)
    for length in (500, 77):  # the lengths are device data: a replay reads the present ones
        args[1][0] = length
        b.lens[0] = length
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        b.check(out)
    assert not torch.equal(out, want)


def test_the_context_scratch_serves_without_a_workspace(gpu):
    b = Batch("q8", 8, 2, 128, lens=[500, 40], nodes=[5, 5])
    want = b.run()
    got = torch.empty_like(want)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s, n, o, m = i32(b.starts), i32(b.lens), i32(b.offsets.tolist()), torch.tensor(b.masks, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    _ffi.call("prana_attention_tree", K.context(), p(b.q), C.byref(b.cache._view), p(s), p(n), p(o), p(m), 2, 10, 5, 8, None, 0, p(got))
    K.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind,n_kv,hd", [("q8", 8, 128), ("f16", 4, 128)])
def test_rows_past_32_bit_offsets(gpu, kind, n_kv, hd):
    positions = (1 << 31) // (n_kv * hd) + 1000  # more than 2^31 elements of K
    cache = K.KvRows.alloc(positions, n_kv, hd, quantized=kind == "q8")
    b = Batch(kind, 2 * n_kv, n_kv, hd, lens=[700], nodes=[6], gap=0)
    first = positions - 706
    for name in ("k", "v", "k_scale", "v_scale"):
        if getattr(cache, name) is not None:
            getattr(cache, name)[first:] = getattr(b.cache, name)[:706]
    b.cache, b.starts = cache, [first]
    b.check()


def test_rows_past_32_bit_offsets_position_by_position(gpu):
    n_kv, hd = 8, 128
    positions = (1 << 31) // (n_kv * hd) + 1000
    k, v = (torch.zeros((positions, n_kv, hd), dtype=torch.int8, device="cuda") for _ in range(2))
    scales = torch.zeros((2, positions, n_kv), device="cuda")
    b = Batch("q8", 2 * n_kv, n_kv, hd, lens=[700], nodes=[6], gap=0)
    cache, first = K.KvRows(k, v, scales[0], scales[1]), positions - 706
    rows, x = torch.arange(706, dtype=torch.int32, device="cuda"), torch.randn(706, n_kv, hd, device="cuda")
    small = K.KvRows.alloc(706, n_kv, hd)
    for c, at in ((small, 0), (cache, first)):
        K.kv_rows_write(c, rows + at, x, x * 2)
    for got, want in zip(K.kv_rows_read(cache, rows + first), K.kv_rows_read(small, rows)):
        assert torch.equal(got, want)
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(cache, name)[first:] = getattr(b.cache, name)[:706]
    b.cache, b.starts = cache, [first]
    b.check()


@pytest.mark.parametrize("kind", ["q8", "f16"])
@pytest.mark.parametrize("hd", [64, 100])
def test_sequences_that_do_not_fit_are_left_out_and_reported(gpu, kind, hd):
    good = Batch(kind, 8, 2, hd, lens=[50, 60, 70], nodes=[3, 3, 3])
    want = good.run()
    K.synchronize()
    for field, b, value in (("starts", 1, -1), ("lens", 1, 10 ** 6), ("lens", 1, -5), ("starts", 1, 2 ** 31 - 1)):
        x = Batch(kind, 8, 2, hd, lens=[50, 60, 70], nodes=[3, 3, 3])
        getattr(x, field)[b] = value
        out = torch.full_like(want, 7.0)
        x.run(out=out)
        with pytest.raises(PranaError, match="PRANA_E_INVALID"):
            K.synchronize()
        assert torch.equal(out[:3], want[:3]) and torch.equal(out[6:], want[6:]) and bool((out[3:6] == 7).all())
    x = Batch(kind, 8, 2, hd, lens=[50, 60, 70], nodes=[3, 3, 3])
    x.max_nodes = 2  # more nodes than the call was told of
    x.run()
    with pytest.raises(PranaError, match="PRANA_E_INVALID"):
        K.synchronize()
    x.max_nodes, x.offsets = 3, np.array([0, 3, 6, 12], np.int32)  # more than q has
    x.run()
    with pytest.raises(PranaError, match="PRANA_E_INVALID"):
        K.synchronize()
    assert torch.equal(good.run(), want)
    K.synchronize()


def test_refusals(gpu):
    b = Batch("q8", 8, 2, 64, lens=[5], nodes=[2])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s, n, o = i32([0]), i32([5]), i32([0, 2])
    q, m = b.q, torch.tensor(b.masks, device="cuda")
    for bad in (lambda: K.attention_tree(q.half(), b.cache, s, n, o, 2, 8), lambda: K.attention_tree(q.cpu(), b.cache, s, n, o, 2, 8),
                lambda: K.attention_tree(q, b.cache, s, n, o, 2, 7), lambda: K.attention_tree(q, b.cache, s, n, o[:1], 2, 8),
                lambda: K.attention_tree(q, b.cache, s, n[:0], o, 2, 8), lambda: K.attention_tree(q, b.cache, s, n, o, 2, 8, m[:1]),
                lambda: K.attention_tree(q, b.cache, s, n, o, 2, 8, m.int()), lambda: K.attention_tree(q[:, ::2], b.cache, s, n, o, 2, 4),
                lambda: K.attention_tree(q, b.cache, s, n, o, 2, 8, m, out=q[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        K.attention_tree(q, b.cache, s.long(), n, o, 2, 8)
    with pytest.raises(PranaError, match="multiple of n_kv_heads"):
        K.attention_tree(q[:, : 7 * 64].contiguous(), b.cache, s, n, o, 2, 7)
    with pytest.raises(PranaError, match="exceed"):
        K.attention_tree(q, b.cache, s, n, o, 65, 8)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    small = torch.empty(512, dtype=torch.uint8, device="cuda")
    with pytest.raises(PranaError, match="bytes"):
        _ffi.call("prana_attention_tree", K.context(), p(q), C.byref(b.cache._view), p(s), p(n), p(o), None, 1, 2, 2, 8, p(small), 16, p(q))
    assert K.attention_tree(q[:0], b.cache, s[:0], n[:0], o[:1], 2, 8).shape == (0, 512)
