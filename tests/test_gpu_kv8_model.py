"""A Whisper context that holds its cross-attention keys and values in 8 bits (owk_context_set_kv8): what is
cached, the decoder's logits over it, and the calls that use it."""
import ctypes as C

import numpy as np
import pytest
import torch

import owk
import whisper_np as O
from test_kv8 import Model

pytestmark = pytest.mark.gpu
LOGIT_RTOL = 1e-3  # as the f16 path's restatement test: f32 re-association through the layers


def _cross(w, st, layer, n, d):
    k, v = np.zeros((n, d), np.uint16), np.zeros((n, d), np.uint16)
    u16 = C.POINTER(C.c_uint16)
    assert w.L.owk_debug_cross(w.ctx, st, 0, layer, k.ctypes.data_as(u16), v.ctypes.data_as(u16)) == n * d
    return k.view(np.float16), v.view(np.float16)


def _encoded(path, pcm, **kw):
    owk.quiet()
    w = owk.Whisper(path, **kw)
    st = w.new_state()
    assert w.L.whisper_pcm_to_mel_with_state(w.ctx, st, owk.fptr(pcm), len(pcm), 1) == 0
    assert w.L.whisper_encode_with_state(w.ctx, st, 0, 1) == 0
    return w, st


def _logits(w, st, tokens, n_past):
    t = (C.c_int32 * len(tokens))(*tokens)
    assert w.L.whisper_decode_with_state(w.ctx, st, t, len(tokens), n_past, 1) == 0
    return np.ctypeslib.as_array(w.L.whisper_get_logits_from_state(st), (len(tokens), w.n_vocab))[-1].copy()


@pytest.mark.parametrize("flash", [True, False])
def test_cached_codes(model_path, clips, flash):
    """Every layer's cross K/V are the f16 context's, rounded to their codes (a last partial block stays f16)."""
    path = model_path("tiny.en")
    hp, _, _ = O.read_model(path)
    n, d, h = hp["n_audio_ctx"], hp["n_text_state"], hp["n_text_head"]
    w, st = _encoded(path, clips["jfk"], flash_attn=flash)
    w8, st8 = _encoded(path, clips["jfk"], flash_attn=flash, kv8=True)
    pad = (n + 255) // 256 * 256 - n if flash else 0
    for layer in range(hp["n_text_layer"]):
        m = Model(1, h, 64, torch.float16)
        x = [torch.from_numpy(a.copy()).view(n, h, 64) for a in _cross(w, st, layer, n, d)]
        zero = torch.zeros((pad, h, 64), dtype=torch.float16)
        m.append(0, 0, *[torch.cat([a, zero]) for a in x])
        got = _cross(w8, st8, layer, n, d)
        for kv, g in zip("kv", got):
            want = m.held(0, kv)[:n].float().half().view(n, d).numpy()
            assert np.array_equal(g, want), (layer, kv)
    w.close()
    w8.close()


class _Decoder8(O.Decoder):
    """The restatement with cross attention as a plain f32 softmax (its pad keys: score 0, value 0)."""

    def step(self, tokens, n_past):
        own = O._one_chunk

        def attend(q, k, v, scale, pad):
            if k.shape[0] != self.hp["n_audio_ctx"]:
                return own(q, k, v, scale, pad)
            s = np.einsum("hd,nhd->hn", q.astype(np.float64), k.astype(np.float64)) * scale
            s = np.concatenate([s, np.zeros((s.shape[0], pad))], 1)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            return np.einsum("hn,nhd->hd", p[:, :k.shape[0]], v.astype(np.float64)).astype(np.float32).astype(np.float16).astype(np.float32)

        O._one_chunk = attend
        try:
            return super().step(tokens, n_past)
        finally:
            O._one_chunk = own


def test_logits(golden, model_path, clips):
    """Prefill and two steps against the restatement over the cached codes."""
    meta, _ = golden
    path = model_path("tiny.en")
    hp, _, t = O.read_model(path)
    w, st = _encoded(path, clips["jfk"], kv8=True)
    cross = [_cross(w, st, layer, hp["n_audio_ctx"], hp["n_text_state"]) for layer in range(hp["n_text_layer"])]
    dec = _Decoder8(hp, t, cross)
    prompt = meta["results"]["tiny.en/jfk/prefill_prompt"]
    n_past, tokens = 0, list(prompt)
    for _ in range(3):
        want, got = dec.step(tokens, n_past), _logits(w, st, tokens, n_past)
        np.testing.assert_allclose(got, want, atol=LOGIT_RTOL * np.abs(want).max(), rtol=0)
        n_past += len(tokens)
        tokens = [int(want.argmax())]
    w.close()


def _ids(segments):
    return [[t[0] for t in s["tokens"]] for s in segments]


@pytest.mark.parametrize("model", ["tiny.en", "l3-mini", "tiny.en q5_0"])
def test_full(model_path, clips, model, tmp_path):
    """whisper_full, greedy and with beams, and a batch: they run, and run the same twice."""
    owk.quiet()
    path = model_path(model.split()[0])
    if model.endswith("q5_0"):
        import owk_synth as S

        S.quantize_q5_0(path, str(tmp_path / "q5.bin"))
        path = str(tmp_path / "q5.bin")
    w = owk.Whisper(path, kv8=True)
    runs = []
    for _ in range(2):
        st = w.new_state()
        p = w.params(0, language="en", temperature_inc=0.0, max_tokens=40)
        assert w.full(st, clips["jfk"], p) == 0
        runs.append(_ids(w.segments(st)))
        w.free_state(st)
    assert runs[0] == runs[1] and sum(map(len, runs[0])) > 0
    st = w.new_state()
    assert w.full(st, clips["jfk"], w.params(1, language="en", temperature_inc=0.0, beam_size=4, max_tokens=40)) == 0
    assert sum(map(len, _ids(w.segments(st)))) > 0
    batch = [w.new_state() for _ in range(3)]
    p = w.params(0, language="en", temperature_inc=0.0, max_tokens=40, initial_prompt=b"a few words before " * 12)
    assert w.full_batch(batch, [clips["jfk"], clips["synth30"], clips["jfk"][:40000]], p) == 0
    assert all(sum(map(len, _ids(w.segments(s)))) > 0 for s in batch)
    w.close()


def test_off_again(golden, model_path, clips):
    """A state that was used in 8 bits and then in f16 gives the f16 results."""
    meta, _ = golden
    owk.quiet()
    w = owk.Whisper(model_path("tiny.en"))
    st = w.new_state()
    p = w.params(0, language="en", temperature_inc=0.0)
    assert w.L.owk_context_set_kv8(w.ctx, 1) == 0
    assert w.full(st, clips["jfk"], p) == 0
    assert w.L.owk_context_set_kv8(w.ctx, 0) == 0
    assert w.full(st, clips["jfk"], p) == 0
    assert _ids(w.segments(st)) == [[t[0] for t in s["tokens"]] for s in meta["results"]["tiny.en/jfk/full/greedy"]["segments"]]
    w.close()


def test_short_audio_context(model_path, clips):
    """audio_ctx below the model's: other numbers of blocks, with and without padded keys."""
    owk.quiet()
    for flash in (True, False):
        w = owk.Whisper(model_path("tiny.en"), kv8=True, flash_attn=flash)
        for ctx in (768, 700, 64, 0):
            st = w.new_state()
            assert w.full(st, clips["jfk"], w.params(0, language="en", temperature_inc=0.0, audio_ctx=ctx, max_tokens=16)) == 0
        w.close()


def test_refused(model_path):
    owk.quiet()
    w = owk.Whisper(model_path("tiny.en"), flash_attn=False, dtw_preset=3)
    assert w.L.owk_context_set_kv8(w.ctx, 1) == -1
    assert w.L.owk_context_set_kv8(w.ctx, 0) == 0
    w.close()
    assert w.L.owk_context_set_kv8(None, 1) == -1
    with pytest.raises(ValueError):
        owk.Whisper(model_path("tiny.en"), flash_attn=False, dtw_preset=3, kv8=True)
