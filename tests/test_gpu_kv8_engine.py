"""A Whisper context that holds its cross-attention keys and values in 8 bits: what its states see of each other, of a change of
the form, and what its logits are beside those over the f16 cache."""
import ctypes as C

import numpy as np
import pytest
import torch

import owk
from test_gpu_kv8_model import _cross, _encoded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv8", [False, True])
def test_rows_of_slots_that_are_not_there(model_path, clips, kv8):
    """owk_debug_cross returns -1 for a slot or layer that is not there."""
    w, st = _encoded(model_path("tiny.en"), clips["jfk"], kv8=kv8)
    k = np.zeros((1500, 384), np.uint16)
    p = k.ctypes.data_as(C.POINTER(C.c_uint16))
    for slot, layer in ((-1, 0), (1, 0), (99, 0), (0, -1), (0, 4)):
        assert w.L.owk_debug_cross(w.ctx, st, slot, layer, p, p) == -1, (slot, layer)
    assert w.L.owk_debug_cross(w.ctx, st, 0, 3, p, p) == k.size
    w.close()
