"""The host side of the cache-row and tree-attention entry points (no GPU):
masks of trees, and refusals that come before any device work."""
import ctypes as C

import pytest
import torch

from prana_b200 import _ffi
from prana_b200 import kernels as K

INVALID = -1


def test_tree_masks():
    assert K.tree_masks([]) == []
    assert K.tree_masks([-1, 0, 0, 2, -1]) == [0b1, 0b11, 0b101, 0b1101, 0b10000]
    chain = K.tree_masks(list(range(-1, 63)))
    assert chain[63] == -1 and chain[62] == (1 << 63) - 1  # signed 64-bit values
    torch.tensor(chain, dtype=torch.int64)


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 0, 5], [-2], list(range(-1, 64))])
def test_tree_masks_refuses(parents):
    with pytest.raises(ValueError):
        K.tree_masks(parents)


def test_rows_must_be_on_a_gpu():
    k = torch.zeros(4, 2, 16, dtype=torch.float16)
    with pytest.raises(ValueError):
        K.KvRows(k, k)


def test_null_arguments_are_codes():
    L = _ffi.lib()
    view = _ffi.KvRowsView()
    assert L.prana_kv_rows_write(None, C.byref(view), None, 1, 0, None, None, 16) == INVALID
    assert L.prana_kv_rows_read(None, C.byref(view), None, 1, 0, None, None) == INVALID
    assert L.prana_kv_rows_move(None, C.byref(view), None, None, None, None, 1, 1) == INVALID
    assert L.prana_attention_tree(None, None, C.byref(view), None, None, None, None, 1, 1, 1, 1, None, 0, None) == INVALID
    assert L.prana_attention_tree_workspace(None, 1, 1, 1, 64, C.byref(C.c_size_t())) == INVALID
    assert b"null" in L.prana_last_error()
