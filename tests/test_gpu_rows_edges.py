"""Cache rows: values and sizes at the edges of f32 and of the entry points.  The
quantiser is restated in test_gpu_rows; comparisons are bit for bit."""
import ctypes as C

import numpy as np
import pytest
import torch
from test_gpu_rows import bits_equal, make_cache, quantise

from prana_b200 import _ffi
from prana_b200 import kernels as K
from prana_b200._ffi import PranaError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["rows", "slice"])
@pytest.mark.parametrize("hd", [64, 128, 100])
def test_write_rows_of_tiny_values(gpu, layout, hd):
    """Scales from subnormal to 1e-30, where 1 / scale or twice that passes f32's range."""
    tops = np.float32([1.5e-45, 1e-42, 1e-40, 1e-38, 3.5e-37, 3.7e-37, 4.2e-37, 5e-37, 6e-37, 7.4e-37, 7.6e-37, 1e-36, 1e-35, 1.2e-34, 1.3e-34, 1e-30])
    rng = np.random.default_rng(hd)
    x = (rng.uniform(-1, 1, (len(tops), 2, hd)).astype(np.float32) * tops[:, None, None]).astype(np.float32)
    x[:, :, 3] = tops[:, None]
    x[:, :, 4] = 0.0
    cache = make_cache(layout, len(tops), 2, hd, True)
    new = torch.from_numpy(x).cuda()
    K.kv_rows_write(cache, torch.arange(len(tops), dtype=torch.int32).cuda(), new, new)
    K.synchronize()
    q, s = quantise(x)
    for got, want in ((cache.k, q), (cache.v, q), (cache.k_scale, s), (cache.v_scale, s)):
        assert bits_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("n_kv", [1, 8])
def test_more_rows_than_a_grid_can_count_are_refused(gpu, n_kv):
    """A last block's threads must not pass 2^31: refused on the host, before any launch."""
    cache = make_cache("rows", 4, n_kv, 16, True)
    rows, x = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, n_kv, 16, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    for n in ((2 ** 31 - 1) // n_kv, (2 ** 31 - 1024) // n_kv):
        with pytest.raises(PranaError, match="too many"):
            _ffi.call("prana_kv_rows_write", K.context(), C.byref(cache._view), p(rows), n, 0, p(x), p(x), n_kv * 16)
        with pytest.raises(PranaError, match="too many"):
            _ffi.call("prana_kv_rows_read", K.context(), C.byref(cache._view), p(rows), n, 0, p(x), p(x))
