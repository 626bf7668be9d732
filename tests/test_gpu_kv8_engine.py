"""A Whisper context that holds its cross-attention keys and values in 8 bits: what its states see of each other, of a change of
the form, and what its logits are beside those over the f16 cache."""
import ctypes as C

import numpy as np
import pytest
import torch

import owk
import whisper_np as O
from test_gpu_kv8_model import _cross, _encoded
from test_kv8 import Model

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


# ---------------------------------------------------------------------------------------------------
# values: several clips, beams, quantised weights, prompts of many rows
# ---------------------------------------------------------------------------------------------------
LOGIT_RTOL = 1e-3  # of the largest logit: f32 re-association through the layers, as the restatement tests have it


def _run(w, pcms, **params):
    """Each clip's logits by the tokens they follow: {(clip, tokens): logits}, from one owk_full_batch call. What is picked is
    not the model's choice but a draw from the tokens before it (a few tokens far above the rest, unevenly spaced for beams), so
    that every run meets the same prefixes."""
    states = [w.new_state() for _ in pcms]
    got = {}

    def cb(ctx, state, tokens, n_tokens, logits, user):
        key = (states.index(state), tuple(tokens[i].id for i in range(n_tokens)))
        x = np.ctypeslib.as_array(logits, shape=(w.n_vocab,))
        got.setdefault(key, x.astype(np.float64))
        rng = np.random.default_rng(key[1])
        x[rng.choice(np.arange(300, 40000), 8, replace=False)] = x[np.isfinite(x)].max() + 60 - np.cumsum(1 + 3 * rng.random(8))

    f = C.CFUNCTYPE(None, C.c_void_p, C.c_void_p, C.POINTER(owk.TokenData), C.c_int, C.POINTER(C.c_float), C.c_void_p)(cb)
    p = w.params(params.pop("strategy", 0), language="en", temperature_inc=0.0, no_timestamps=True, **params)
    p.logits_filter_callback = C.cast(f, C.c_void_p)
    assert w.full_batch(states, pcms, p) == 0
    return states, got


def _apart(a, b):
    """The largest difference of two rows of logits, of the largest of them."""
    ok = np.isfinite(a) & np.isfinite(b)
    assert ok.sum() > 1000
    return np.abs(a[ok] - b[ok]).max() / np.abs(b[ok]).max()


def _model(model_path, tmp_path, model):
    path = model_path(model.split()[0])
    if model.endswith("q5_0"):
        import owk_synth as S

        S.quantize_q5_0(path, str(tmp_path / "q5.bin"))
        path = str(tmp_path / "q5.bin")
    return path


@pytest.mark.parametrize("model", ["tiny.en", "l3-mini", "tiny.en q5_0"])
@pytest.mark.parametrize("beams", [0, 4])
def test_clips_of_a_batch(model_path, clips, tmp_path, model, beams):
    """Each clip of a batch has the logits that it has alone, after every prefix; and not another clip's.
    With quantised weights a batch differs from a clip alone in either form of the cache (activations are rounded to 1/127 of
    their block's largest, so an f32 difference can move one by a step): there a clip's logits have to be nearer to its own than to
    any other clip's, and the 8-bit cache's to the f16 cache's of the same clip."""
    owk.quiet()
    path = _model(model_path, tmp_path, model)
    quant = model.endswith("q5_0")
    w = owk.Whisper(path, kv8=True)
    pcms = [clips["synth30"], clips["jfk"], clips["jfk"][:40000], clips["synth30"][:200000]]
    kw = dict(max_tokens=12, initial_prompt=b"a few words before " * 12)
    if beams:
        kw |= dict(strategy=1, beam_size=beams)
    _, batch = _run(w, pcms, **kw)
    runs = [_run(w, [pcm], **kw)[1] for pcm in pcms]
    if quant:
        w16 = owk.Whisper(path)
        _, batch16 = _run(w16, pcms, **kw)
        w16.close()
    for c, alone in enumerate(runs):
        both = [t for _, t in alone]
        assert len(both) >= 12 and all((c, t) in batch for t in both), c
        met = 0
        for t in both:
            others = [_apart(batch[o, t], alone[0, t]) for o in range(len(pcms)) if o != c and (o, t) in batch]
            mine = _apart(batch[c, t], alone[0, t])
            met += len(others)
            if quant:
                assert mine < min(others, default=np.inf), (c, t)
                others16 = [_apart(batch16[o, t], batch[c, t]) for o in range(len(pcms)) if o != c and (o, t) in batch16]
                assert _apart(batch16[c, t], batch[c, t]) < min(others16, default=np.inf), (c, t)
            else:
                assert mine <= LOGIT_RTOL, (c, t, mine)
                assert min(others, default=np.inf) > 8 * LOGIT_RTOL, (c, t)
        assert met > 0
    w.close()


@pytest.mark.parametrize("model", ["tiny.en", "l3-mini"])
def test_codes_of_every_slot(model_path, clips, model):
    """Cross K/V of all slots of a batch: the f16 context's, rounded to their codes."""
    owk.quiet()
    path = model_path(model)
    hp, _, _ = O.read_model(path)
    n, d, h = hp["n_audio_ctx"], hp["n_text_state"], hp["n_text_head"]
    pcms = [clips["synth30"], clips["jfk"], clips["jfk"][:40000]]
    w, w8 = owk.Whisper(path), owk.Whisper(path, kv8=True)
    states, _ = _run(w, pcms, max_tokens=2)
    states8, _ = _run(w8, pcms, max_tokens=2)
    u16 = C.POINTER(C.c_uint16)
    zero = torch.zeros(((n + 255) // 256 * 256 - n, h, 64), dtype=torch.float16)
    for slot in range(3):
        for layer in range(hp["n_text_layer"]):
            x, y = np.zeros((2, n, d), np.uint16), np.zeros((2, n, d), np.uint16)
            for ww, st, a in ((w, states[0], x), (w8, states8[0], y)):
                assert ww.L.owk_debug_cross(ww.ctx, st, slot, layer, a[0].ctypes.data_as(u16), a[1].ctypes.data_as(u16)) == n * d
            m = Model(1, h, 64, torch.float16)
            m.append(0, 0, *[torch.cat([torch.from_numpy(a.view(np.float16)).view(n, h, 64), zero]) for a in x])
            for kv, g in zip("kv", y):
                want = m.held(0, kv)[:n].float().half().view(n, d).numpy()
                assert np.array_equal(g.view(np.float16), want), (slot, layer, kv)
    w.close()
    w8.close()


class _Decoder8(O.Decoder):
    """The restatement with cross attention as a plain softmax in 64 bits, also for prompts of many rows (their other attention
    works on heads x rows x dim; pad keys: score 0, value 0)."""

    def step(self, tokens, n_past):
        own = O._one_chunk, O._flash_tiled
        n_audio = self.hp["n_audio_ctx"]

        def plain(q, k, v, scale, pad):  # q [h, d], k / v [n, h, d]
            s = np.einsum("hd,nhd->hn", q.astype(np.float64), k.astype(np.float64)) * scale
            s = np.concatenate([s, np.zeros((s.shape[0], pad))], 1)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            return np.einsum("hn,nhd->hd", p[:, :k.shape[0]], v.astype(np.float64)).astype(np.float32).astype(np.float16).astype(np.float32)

        def one_chunk(q, k, v, scale, pad):
            return plain(q, k, v, scale, pad) if k.shape[0] == n_audio else own[0](q, k, v, scale, pad)

        def tiled(q, k, v, scale, pad):
            if k.shape[1] != n_audio:
                return own[1](q, k, v, scale, pad)
            return plain(q[:, 0], k.transpose(1, 0, 2), v.transpose(1, 0, 2), scale, pad)

        O._one_chunk, O._flash_tiled = one_chunk, tiled
        try:
            return super().step(tokens, n_past)
        finally:
            O._one_chunk, O._flash_tiled = own


def _prompt(golden, n):
    meta, _ = golden
    start = [int(x) for x in meta["results"]["tiny.en/jfk/prefill_prompt"]]
    gen = np.random.default_rng(5)
    return [int(x) for x in gen.integers(200, 40000, n - len(start))] + start


@pytest.mark.parametrize("rows", [32, 1 << 30])
def test_logits_of_a_long_prompt(golden, model_path, clips, rows):
    """A prompt of 48 rows in both forms of attention, and a step behind it, against the restatement over the cached codes."""
    path = model_path("tiny.en")
    hp, _, t = O.read_model(path)
    tokens = _prompt(golden, 48)
    owk.load().owk_debug_kv8_set_many_rows(rows)
    try:
        w, st = _encoded(path, clips["jfk"], kv8=True)
        cross = [_cross(w, st, layer, hp["n_audio_ctx"], hp["n_text_state"]) for layer in range(hp["n_text_layer"])]
        dec = _Decoder8(hp, t, cross)
        for toks, past in ((tokens, 0), ([tokens[-1]], 48)):
            want = dec.step(toks, past)
            assert _decode(w, st, toks, past) == 0
            np.testing.assert_allclose(_last_logits(w, st, len(toks)), want, atol=LOGIT_RTOL * np.abs(want).max(), rtol=0)
        w.close()
    finally:
        owk.load().owk_debug_kv8_set_many_rows(0)


def test_logits_beside_the_f16_cache(golden, model_path, clips):
    """The logits over the 8-bit cache are as far from those over the f16 cache as the codes make them: the restatements of both
    paths over both caches say how far that is, and each run is within its own bound of its restatement."""
    path = model_path("tiny.en")
    hp, _, t = O.read_model(path)
    n, d = hp["n_audio_ctx"], hp["n_text_state"]
    tokens = _prompt(golden, 40)
    runs, decs = [], []
    for kv8 in (False, True):
        w, st = _encoded(path, clips["jfk"], kv8=kv8)
        decs.append((_Decoder8 if kv8 else O.Decoder)(hp, t, [_cross(w, st, layer, n, d) for layer in range(hp["n_text_layer"])]))
        runs.append((w, st))
    for toks, past in ((tokens, 0), ([tokens[-1]], 40), ([tokens[-2]], 41)):
        o16, o8 = (x.step(toks, past) for x in decs)
        got = []
        for w, st in runs:
            assert _decode(w, st, toks, past) == 0
            got.append(_last_logits(w, st, len(toks)))
        bound = np.abs(o8 - o16).max() + LOGIT_RTOL * (np.abs(o16).max() + np.abs(o8).max())
        assert np.abs(got[1] - got[0]).max() <= bound, (past, np.abs(got[1] - got[0]).max(), bound)
    for w, _ in runs:
        w.close()
