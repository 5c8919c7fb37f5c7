"""attention_tree: rows of the result that no sequence fills, and a call told of no nodes."""
import pytest
import torch
from test_gpu_tree import Batch

from prana_b200 import kernels as K
from prana_b200._ffi import PranaError

pytestmark = pytest.mark.gpu


def test_nodes_without_max_nodes_are_refused(gpu):
    b = Batch("q8", 8, 2, 64, lens=[50], nodes=[3])
    b.max_nodes = 0
    with pytest.raises(PranaError, match="max_nodes is 0"):
        b.run()
    assert K.attention_tree(b.q[:0], b.cache, *(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 1, 2)), 0, 8).shape == (0, 512)
