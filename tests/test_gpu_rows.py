"""Cache rows by index on the GPU: quantising write, read back, and the move of
accepted branches, against a numpy restatement.  Everything here is integers,
copies or one IEEE operation per value, so every comparison is bit for bit."""
import numpy as np
import pytest
import torch

from prana_b200 import kernels as K
from prana_b200._ffi import PranaError

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 16), (3, 2, 64), (37, 8, 128), (5, 6, 48), (9, 3, 96), (4, 1, 256), (6, 2, 100), (2, 5, 7), (33, 4, 32)]


def quantise(x):
    """quantize_q8 over each head row of f32 x [n, n_kv, hd]: (int8, f32 scales)."""
    with np.errstate(all="ignore"):
        amax = np.fmax.reduce(np.abs(x), axis=-1, initial=np.float32(0))
        scale = np.where(amax > 0, amax / np.float32(127), np.float32(1)).astype(np.float32)
        t = x * (np.float32(1) / scale)[..., None]
        r = np.copysign(np.floor(np.abs(t.astype(np.float64)) + 0.5), t)
        return np.where(np.isnan(r), 0, np.clip(r, -127, 127)).astype(np.int8), scale


def make_cache(layout, positions, n_kv, hd, quantized, seed=0):
    """A cache filled with values, in one of several memory layouts."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def tensor():
        if quantized:
            x = torch.randint(-127, 128, (positions, n_kv, hd), generator=g, device="cuda", dtype=torch.int8)
        else:
            x = torch.randn((positions, n_kv, hd), generator=g, device="cuda").half()
        if layout == "heads":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "slice":  # odd strides and an unaligned start
            wide = torch.zeros((positions, n_kv, hd + 5), dtype=x.dtype, device="cuda")
            wide[:, :, 3:3 + hd] = x
            return wide[:, :, 3:3 + hd]
        return x

    k, v = tensor(), tensor()
    if not quantized:
        return K.KvRows(k, v)
    s = torch.rand((2, n_kv, positions), generator=g, device="cuda") + 0.5
    if layout == "heads":
        return K.KvRows(k, v, s[0].t(), s[1].t())
    return K.KvRows(k, v, s[0].t().contiguous(), s[1].t().contiguous())


def host(cache):
    return [None if t is None else t.cpu().numpy().copy() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def bits_equal(a, b):
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    both_nan = np.isnan(a) & np.isnan(b) if a.dtype.kind == "f" else np.zeros(a.shape, bool)
    return a.dtype == b.dtype and a.shape == b.shape and bool(np.all((a == b) | both_nan))


def rows_for(n, positions, seed, skip=True):
    rng = np.random.default_rng(seed)
    rows = rng.permutation(positions)[:n].astype(np.int32)
    if skip and n > 2:
        rows[n // 2] = -1
    return rows


@pytest.mark.parametrize("layout", ["rows", "heads", "slice"])
@pytest.mark.parametrize("src", [torch.float32, torch.float16])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("n,n_kv,hd", SIZES)
def test_write_matches_numpy(gpu, n, n_kv, hd, quantized, src, layout):
    positions = n + 11
    cache = make_cache(layout, positions, n_kv, hd, quantized)
    want = host(cache)
    rng = np.random.default_rng(n * 7 + hd)
    new = [torch.from_numpy(rng.standard_normal((n, n_kv, hd)).astype(np.float32) * 3).to(src) for _ in range(2)]
    new[0][0] = 0.0  # an all-zero row: scale 1
    rows = rows_for(n, positions, seed=hd)
    K.kv_rows_write(cache, torch.from_numpy(rows).cuda(), new[0].cuda(), new[1].cuda())
    K.synchronize()
    for i, row in enumerate(rows):
        if row < 0:
            continue
        for j in range(2):
            x = new[j][i].float().numpy()
            if quantized:
                want[j][row], want[2 + j][row] = quantise(x)
            else:
                want[j][row] = x.astype(np.float16)
    for got, ref in zip(host(cache), want):
        assert ref is None or bits_equal(got, ref)


@pytest.mark.parametrize("n,n_kv,hd", [(5, 2, 64), (3, 8, 128), (3, 2, 100)])
def test_write_values_that_are_not_numbers(gpu, n, n_kv, hd):
    cache = make_cache("rows", n + 3, n_kv, hd, True)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((n, n_kv, hd)).astype(np.float32)
    x[0, 0, 1] = np.nan           # a NaN becomes 0, the rest of its row keeps its scale
    x[0, 1] = np.nan              # nothing but NaN: scale 1
    x[1, 0, 2] = np.inf           # an infinity: infinite scale, the row reads back as NaN
    x[2, 0] = 1e-42               # subnormal values
    x[2, 1] *= np.float32(1e38)   # near the largest
    K.kv_rows_write(cache, torch.arange(n, dtype=torch.int32).cuda(), torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda())
    back, _ = K.kv_rows_read(cache, torch.arange(n, dtype=torch.int32).cuda())
    K.synchronize()
    q, s = quantise(x)
    assert bits_equal(cache.k[:n].cpu().numpy(), q) and bits_equal(cache.v[:n].cpu().numpy(), q)
    assert bits_equal(cache.k_scale[:n].cpu().numpy(), s)
    assert torch.isnan(back[1, 0]).all() and torch.isfinite(back[0]).all()


def test_write_takes_strided_and_flat_sources(gpu):
    n, n_kv, hd = 12, 2, 64
    cache = make_cache("rows", 40, n_kv, hd, True)
    ref = make_cache("rows", 40, n_kv, hd, True)
    wide = torch.randn(n, 3, n_kv * hd + 1, device="cuda")  # Q|K|V-like rows, unaligned
    k, v = wide[:, 1, 1:], wide[:, 2, 1:]
    rows = torch.arange(5, 5 + n, dtype=torch.int32, device="cuda")
    K.kv_rows_write(cache, rows, k, v)
    K.kv_rows_write(ref, rows, k.contiguous().view(n, n_kv, hd), v.contiguous().view(n, n_kv, hd))
    K.synchronize()
    for a, b in zip(host(cache), host(ref)):
        assert bits_equal(a, b)


@pytest.mark.parametrize("layout", ["rows", "heads", "slice"])
@pytest.mark.parametrize("dst", [torch.float32, torch.float16])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("n,n_kv,hd", SIZES)
def test_read_matches_numpy(gpu, n, n_kv, hd, quantized, dst, layout):
    positions = n + 11
    cache = make_cache(layout, positions, n_kv, hd, quantized)
    rows = rows_for(n, positions, seed=hd + 1)
    got = K.kv_rows_read(cache, torch.from_numpy(rows).cuda(), dst)
    K.synchronize()
    h = host(cache)
    for j in range(2):
        want = h[j][np.maximum(rows, 0)].astype(np.float32)
        if quantized:
            want = want * h[2 + j][np.maximum(rows, 0)][..., None]
        want[rows < 0] = 0
        assert bits_equal(got[j].cpu().numpy(), want.astype(np.float32 if dst is torch.float32 else np.float16))


@pytest.mark.parametrize("layout", ["rows", "heads", "slice"])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("n_seq,nodes,n_kv,hd", [(1, 1, 1, 16), (3, 8, 2, 64), (7, 64, 8, 128), (4, 64, 1, 256), (5, 33, 2, 100), (2, 5, 3, 7)])
def test_move_matches_numpy(gpu, n_seq, nodes, n_kv, hd, quantized, layout):
    rng = np.random.default_rng(nodes)
    lens = rng.integers(0, 20, n_seq).astype(np.int32)
    starts = np.cumsum(np.concatenate([[0], lens[:-1] + nodes + 2])).astype(np.int32)
    positions = int(starts[-1] + lens[-1] + nodes)
    cache = make_cache(layout, positions, n_kv, hd, quantized)
    want = host(cache)
    path = np.zeros((n_seq, nodes), np.int32)
    counts = rng.integers(0, nodes + 1, n_seq).astype(np.int32)
    for b in range(n_seq):
        path[b, : counts[b]] = np.sort(rng.permutation(nodes)[: counts[b]])
        if b == n_seq - 1:  # any order: the rows move at once
            path[b, : counts[b]] = rng.permutation(nodes)[: counts[b]]
        base = starts[b] + lens[b]
        for w in want:
            if w is not None:
                w[base:base + counts[b]] = w[base + path[b, : counts[b]]]
    K.kv_rows_move(cache, *(torch.from_numpy(x).cuda() for x in (starts, lens, path, counts)))
    K.synchronize()
    for got, ref in zip(host(cache), want):
        assert ref is None or bits_equal(got, ref)


def test_empty_calls(gpu):
    cache = make_cache("rows", 4, 2, 64, True)
    before = host(cache)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    K.kv_rows_write(cache, none, torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"))
    k, v = K.kv_rows_read(cache, none)
    K.kv_rows_move(cache, none, none, none.view(0, 0), none)
    K.synchronize()
    assert k.shape == (0, 2, 64) and v.shape == (0, 2, 64)
    for a, b in zip(host(cache), before):
        assert bits_equal(a, b)


def test_rows_past_32_bit_offsets(gpu):
    positions, n_kv, hd = (1 << 31) // (8 * 128) + 4099, 8, 128  # more than 2^31 bytes of K
    cache = K.KvRows.alloc(positions, n_kv, hd)
    x = torch.randn(3, n_kv, hd, device="cuda")
    rows = torch.tensor([positions - 1, 5, positions - 4098], dtype=torch.int32, device="cuda")
    K.kv_rows_write(cache, rows, x, x * 2)
    k, v = K.kv_rows_read(cache, rows)
    start = torch.tensor([positions - 4098], dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    path, one = torch.full((1, 1), 4097, dtype=torch.int32, device="cuda"), zero + 1
    K.kv_rows_move(cache, start, zero, path, one)
    K.synchronize()
    q, s = quantise(x.cpu().numpy())
    assert bits_equal(k.cpu().numpy(), q.astype(np.float32) * s[..., None])
    assert bits_equal(cache.k[positions - 1].cpu().numpy(), q[0]) and bits_equal(cache.k[positions - 4098].cpu().numpy(), q[0])
    assert int(cache.k[5].abs().max()) == 127 and int(cache.k[6].abs().max()) == 0


def test_rows_outside_the_cache_are_left_out_and_reported(gpu):
    cache = make_cache("rows", 8, 2, 64, True)
    before = host(cache)
    x = torch.randn(2, 2, 64, device="cuda")
    bad = torch.tensor([8, -7], dtype=torch.int32, device="cuda")
    K.kv_rows_write(cache, bad, x, x)
    with pytest.raises(PranaError, match="PRANA_E_INVALID"):
        K.synchronize()
    k, _ = K.kv_rows_read(cache, bad)
    with pytest.raises(PranaError, match="PRANA_E_INVALID"):
        K.synchronize()
    assert int(k.count_nonzero()) == 0
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for starts, lens, path, counts in [((0,), (7,), (0, 1), (2,)), ((-1,), (2,), (0, 1), (2,)), ((0,), (2,), (0, 6), (2,)), ((0,), (2,), (0, -1), (2,)), ((0,), (2,), (0, 1), (3,))]:
        p = i32(*path).view(1, 2)
        if path == (0, 1):
            p = i32(1, 0).view(1, 2)
        K.kv_rows_move(cache, i32(*starts), i32(*lens), p, i32(*counts))
        with pytest.raises(PranaError, match="PRANA_E_INVALID"):
            K.synchronize()
    K.synchronize()  # reported once
    for a, b in zip(host(cache), before):
        assert bits_equal(a, b)


def test_refusals(gpu):
    cache = make_cache("rows", 8, 2, 64, True)
    k, s = cache.k, cache.k_scale
    rows = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.randn(2, 2, 64, device="cuda")
    for bad in (lambda: K.KvRows(k, k), lambda: K.KvRows(k, k[:4], s, s), lambda: K.KvRows(k, k, s[:4], s),
                lambda: K.KvRows(k.half(), k.half(), s, s), lambda: K.KvRows(k.transpose(1, 2), k.transpose(1, 2), s, s),
                lambda: K.KvRows(k, k, s, s.cpu()),
                lambda: K.kv_rows_write(cache, rows, x[:1], x[:1]), lambda: K.kv_rows_write(cache, rows, x, x.half()),
                lambda: K.kv_rows_write(cache, rows, x.cpu(), x.cpu()), lambda: K.kv_rows_write(cache, rows.cpu(), x, x),
                lambda: K.kv_rows_move(cache, rows, rows, rows, rows), lambda: K.kv_rows_move(cache, rows, rows, rows.view(1, 2), rows)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: K.KvRows(k.float(), k.float()), lambda: K.KvRows(k, k, s.half(), s.half()),
                lambda: K.kv_rows_write(cache, rows.long(), x, x), lambda: K.kv_rows_write(cache, rows, x.double(), x.double()),
                lambda: K.kv_rows_read(cache, rows, torch.bfloat16)):
        with pytest.raises(TypeError):
            bad()
    wide = torch.zeros(4, 1, 257, dtype=torch.float16, device="cuda")
    with pytest.raises(PranaError, match="head_dim"):
        K.kv_rows_read(K.KvRows(wide, wide), rows)
    with pytest.raises(PranaError, match="exceeds 64"):
        K.kv_rows_move(cache, rows, rows, torch.zeros(2, 65, dtype=torch.int32, device="cuda"), rows)
