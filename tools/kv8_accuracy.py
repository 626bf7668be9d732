"""How far a model's logits move with its cross keys and values in 8 bits: bench.py's clips, greedy, a fixed number of tokens.

  python tools/kv8_accuracy.py [--model large-v3] [--clips 8] [--tokens 220]

Runs the clips over the f16 cache and keeps every step's logits; runs them again, forced onto the same tokens, over the 8-bit cache,
and once more over the f16 cache in two batches of half the clips (what another batch alone moves). Prints, for both: the largest
and the mean root-mean-square difference of a step's logits (of the standard deviation of the step's logits), and how many
steps pick the same token."""
import argparse
import ctypes as C
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "open-whisper-kit_amd", "python"))

import numpy as np  # noqa: E402

import owk  # noqa: E402
import owk_synth as S  # noqa: E402


def run(w, pcms, n_tokens, forced=None):
    """[clip][step] logits of a greedy run (EOT suppressed), on the given tokens if there are any."""
    states = [w.new_state() for _ in pcms]
    eot = w.L.whisper_token_eot(w.ctx)
    kept = [[] for _ in pcms]

    def cb(ctx, state, tokens, n, logits, user):
        c = states.index(state)
        x = np.ctypeslib.as_array(logits, shape=(w.n_vocab,))
        kept[c].append(x.astype(np.float32))
        kept[c][-1][eot] = -np.inf
        if forced is not None and n < len(forced[c]):
            x[forced[c][n]] = float(x[np.isfinite(x)].max()) + 40.0

    f = C.CFUNCTYPE(None, C.c_void_p, C.c_void_p, C.POINTER(owk.TokenData), C.c_int, C.POINTER(C.c_float), C.c_void_p)(cb)
    p = w.params(0, language="en", temperature_inc=0.0, no_timestamps=True, max_tokens=n_tokens - 1)
    p.logits_filter_callback = C.cast(f, C.c_void_p)
    if w.full_batch(states, pcms, p, suppress_eot=True) != 0:
        raise RuntimeError("owk_full_batch failed")
    ids = [[t[0] for s in w.segments(st) for t in s["tokens"]] for st in states]
    for st in states:
        w.L.whisper_free_state(st)
    w._states = [x for x in w._states if x not in states]
    return kept, ids


def compare(a, b):
    rms, worst, same, n = [], 0.0, 0, 0
    for x, y in zip(a, b):
        for u, v in zip(x, y):
            ok = np.isfinite(u) & np.isfinite(v)
            d = u[ok].astype(np.float64) - v[ok]
            rms.append(float(np.sqrt((d * d).mean()) / v[ok].astype(np.float64).std()))
            worst = max(worst, rms[-1])
            same += int(np.argmax(u) == np.argmax(v))
            n += 1
    return {"steps": n, "rms_mean": round(float(np.mean(rms)), 6), "rms_worst": round(worst, 6), "same_pick": same}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--model", default="large-v3")
    ap.add_argument("--clips", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=220)
    args = ap.parse_args()
    owk.quiet()
    path = S.ensure_model(args.model, cache_dir=os.environ.get("OWK_MODEL_CACHE", "/tmp/owk_models"))
    pcms = [S.synth_audio(480000, seed) for seed in range(args.clips)]
    w = owk.Whisper(path)
    want, ids = run(w, pcms, args.tokens)
    print(f"f16 cache: {sum(map(len, want))} steps", file=sys.stderr, flush=True)
    half = args.clips // 2
    other = run(w, pcms[:half], args.tokens, ids[:half])[0] + run(w, pcms[half:], args.tokens, ids[half:])[0]
    w.close()
    w = owk.Whisper(path, kv8=True)
    got, _ = run(w, pcms, args.tokens, ids)
    w.close()
    print(json.dumps({"model": args.model, "clips": args.clips, "tokens": args.tokens,
                      "kv8_against_f16": compare(got, want), "f16_in_half_batches": compare(other, want)}), flush=True)


if __name__ == "__main__":
    main()
