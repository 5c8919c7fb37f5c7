"""attention_tree: rows of the result that no sequence fills, and a call told of no nodes."""
import pytest
import torch
from test_gpu_tree import Batch

from prana_b200 import kernels as K
from prana_b200._ffi import PranaError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 100])
@pytest.mark.parametrize("kind", ["q8", "f16"])
def test_rows_of_no_sequence_stay_as_they_are(gpu, kind, hd):
    b = Batch(kind, 8, 2, hd, lens=[50, 300], nodes=[3, 4])
    want = b.run().clone()
    b.q = torch.cat((b.q, b.q))  # more rows than the sequences have nodes
    b.masks = b.masks + b.masks
    out = torch.full((14, 8 * hd), 7.0, device="cuda")
    b.run(out=out)
    K.synchronize()
    assert torch.equal(out[:7], want) and bool((out[7:] == 7).all())


def test_nodes_without_max_nodes_are_refused(gpu):
    b = Batch("q8", 8, 2, 64, lens=[50], nodes=[3])
    b.max_nodes = 0
    with pytest.raises(PranaError, match="max_nodes is 0"):
        b.run()
    assert K.attention_tree(b.q[:0], b.cache, *(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 1, 2)), 0, 8).shape == (0, 512)
