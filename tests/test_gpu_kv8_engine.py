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


def _decode(w, st, tokens, n_past):
    t = (C.c_int32 * len(tokens))(*tokens)
    return w.L.whisper_decode_with_state(w.ctx, st, t, len(tokens), n_past, 1)


def _last_logits(w, st, n):
    return np.ctypeslib.as_array(w.L.whisper_get_logits_from_state(st), (n, w.n_vocab))[-1].copy()


@pytest.mark.parametrize("first", [False, True])
def test_change_of_form_between_calls(golden, model_path, clips, first):
    """What was encoded in the other form is refused, not read; encoded again, the state goes on with its decoded tokens."""
    meta, _ = golden
    prompt = meta["results"]["tiny.en/jfk/prefill_prompt"]
    w, st = _encoded(model_path("tiny.en"), clips["jfk"], kv8=first)
    assert _decode(w, st, prompt, 0) == 0
    assert w.L.owk_context_set_kv8(w.ctx, 0 if first else 1) == 0
    assert _decode(w, st, [int(prompt[-1])], len(prompt)) != 0
    assert _decode(w, st, prompt, 0) != 0
    assert w.L.whisper_encode_with_state(w.ctx, st, 0, 1) == 0
    assert _decode(w, st, [int(prompt[-1])], len(prompt)) == 0
    got = _last_logits(w, st, 1)
    assert w.L.owk_context_set_kv8(w.ctx, 1 if first else 0) == 0
    assert w.L.whisper_encode_with_state(w.ctx, st, 0, 1) == 0
    assert _decode(w, st, [int(prompt[-1])], len(prompt)) == 0
    back = _last_logits(w, st, 1)
    fresh, stf = _encoded(model_path("tiny.en"), clips["jfk"], kv8=first)
    assert _decode(fresh, stf, prompt, 0) == 0 and _decode(fresh, stf, [int(prompt[-1])], len(prompt)) == 0
    want = _last_logits(fresh, stf, 1)
    # back in the first form: the same keys, values, self-attention cache and kernels
    assert np.array_equal(back, want)
    # in the other form near it, and not what an empty self-attention cache gives
    assert _decode(fresh, stf, [int(prompt[-1])], 0) == 0
    alone = _last_logits(fresh, stf, 1)
    assert np.abs(got - want).max() < 0.25 * np.abs(alone - want).max()
    w.close()
    fresh.close()
