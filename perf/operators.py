"""The 8-bit key/value cache: filling it, attending over it, reading it back.

A sequence's keys and values are held in blocks of 64 tokens. A complete block holds, for each
key/value head, 64 * D signed 8-bit codes and one scale s = max|x| / 127 (keys and values apart); a
code c stands for c * s. The last, incomplete block (the tail) stays in the 16-bit type it came in.

  append  n new tokens a sequence; the blocks they touch are then read back in 16 bits
  attend  attention of new query rows over what the cache holds (cross attention: every row sees
          every key; causal: a row sees the keys up to its own place)
  step    append and causal attention of the same tokens: one layer of a decoding step or a chunk

Layouts: k codes [block][head][64][D], v codes [block][head][D][64], scales [block][head],
k tail [sequence][head][64][D], v tail [sequence][head][D][64]; `table` names the blocks of a sequence.
`lens` counts the tokens that are in the cache before the call.
"""
import math
import random
import sys

import torch

own = False

BLOCK = 64
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, dtype, dim, heads, group, seqs, new, hist, causal=False, paged=False):
    return {"name": name, "op": op, "dtype": dtype, "dim": dim, "heads": heads, "group": group, "seqs": seqs,
            "new_lo": new[0], "new_hi": new[1], "hist_lo": hist[0], "hist_hi": hist[1], "causal": causal, "paged": paged}


def listed():
    return [
        # the key and value of one decoded token for each of 32 streams (20 heads of 64): a prompt of five tokens to a full text context;
        # two of the streams complete a block
        _case("append token", "append", "f16", 64, 20, 1, 32, (1, 1), (5, 447)),
        # the cross keys and values of 32 encoded clips, one layer: 1500 frames each into an empty cache
        _case("append clips", "append", "f16", 64, 20, 1, 32, (1500, 1500), (0, 0)),
        # chunks of differing length joined into one call, paged cache, grouped heads
        _case("append ragged", "append", "bf16", 128, 8, 4, 13, (1, 700), (0, 900), paged=True),
        # cross attention of one decoding step, one clip: latency
        _case("cross 1 clip", "attend", "f16", 64, 20, 1, 1, (1, 1), (1500, 1500)),
        # the same for the batch of 32 clips
        _case("cross 32 clips", "attend", "f16", 64, 20, 1, 32, (1, 1), (1500, 1500)),
        # 8 clips with 5 beams each: five rows share one clip's keys
        _case("cross beams", "attend", "f16", 64, 20, 1, 8, (5, 5), (1500, 1500)),
        # the prompt pass of 32 clips: 1 to 224 rows each (half the text context at most), joined
        _case("cross prompts", "attend", "f16", 64, 20, 1, 32, (1, 224), (1500, 1500)),
        # one token for each of 16 long streams of very different length, grouped heads, paged
        _case("long streams", "attend", "bf16", 128, 8, 4, 16, (1, 1), (900, 33000), causal=True, paged=True),
        # one very long stream and few heads: the work has to be split along the keys
        _case("one long stream", "attend", "bf16", 128, 4, 8, 1, (1, 1), (98765, 98765), causal=True, paged=True),
        # chunks of a long prompt over what came before
        _case("chunks", "attend", "bf16", 128, 8, 4, 4, (301, 1024), (0, 8000), causal=True, paged=True),
        # one layer of a decoding step: the token goes in, then it attends; 6 heads, one stream
        _case("step 1 stream", "step", "f16", 64, 6, 1, 1, (1, 1), (0, 447), causal=True),
        # the same for 48 streams of 16 heads
        _case("step 48 streams", "step", "f16", 64, 16, 1, 48, (1, 1), (5, 447), causal=True),
    ]


def _counts(case, rng=None):
    """New tokens and history of each sequence: the same numbers for every seed, in an order of its own."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    got = [[r.randint(case[c + "_lo"], case[c + "_hi"]) for _ in range(case["seqs"])] for c in ("new", "hist")]
    if rng is not None:
        rng.shuffle(got[0])
        rng.shuffle(got[1])
    return got


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())

    def log(lo, hi):
        return min(hi, int(lo * math.exp(rng.random() * math.log((hi + 1) / lo))))

    while True:
        op = rng.choice(["append", "attend", "attend", "step"])
        dim = rng.choice([64, 128])
        heads, group = rng.randint(1, 20), rng.choice([1, 1, 2, 3, 4, 5, 8])
        seqs = log(1, 48)
        new = log(1, 1500) if rng.random() < 0.6 else 1
        hist = log(1, 60000 if seqs <= 4 else 6000) - 1
        causal = op == "step" or rng.random() < 0.5
        ragged = rng.random() < 0.5 and new > 1
        hist = hist if causal else max(1, hist)
        case = _case("", op, rng.choice(["f16", "bf16"]), dim, heads, group, seqs, (1 if ragged else new, new),
                     (max(int(hist * rng.choice([0, 0.3, 1])), min(hist, 1)), hist), causal, rng.random() < 0.5)
        if _cost(case) <= most and seqs * (hist + new) * heads * dim <= 1 << 28:
            del case["name"]
            return case


def work(case):
    h, d, g = case["heads"], case["dim"], case["group"]
    new, hist = _counts(case)
    token = sum(new) * h * d * 2  # the new keys and values
    code = 1 + 4 / (BLOCK * d)    # a code and its share of the scale
    append = token * (2 + code)
    if case["op"] == "append":  # and reading back the touched blocks
        return {"bytes": append + token * (code + 2), "flops": 4 * token}
    held = sum(hist) + (sum(new) if case["causal"] else 0)
    pairs = sum(n * (x + (n + 1) / 2 if case["causal"] else x) for n, x in zip(new, hist))
    attend = 2 * held * h * d * code + 2 * sum(new) * h * g * d * 2
    return {"bytes": attend + (append if case["op"] == "step" else 0), "flops": 4 * pairs * h * g * d}


# ---------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------
def _window(state, kv, new, lens, off, n_new, blocks):
    """The tokens of the `blocks` blocks that an append touches: [b, blocks, 64, h, d], zeros behind the last."""
    tail = state[kv + "_tail"]
    base = lens // BLOCK * BLOCK
    pos = base[:, None] + torch.arange(blocks * BLOCK, device=lens.device)
    if kv == "v":
        tail = tail.transpose(2, 3)
    old = tail.permute(0, 2, 1, 3)[:, (pos[0] - base[0]) % BLOCK]
    at = (pos - lens[:, None]).clamp(min=0)
    row = (off[:-1, None] + at).clamp(max=max(0, new.shape[0] - 1))
    x = torch.where((pos < lens[:, None])[..., None, None], old, new[row])
    x = torch.where((pos < (lens + n_new)[:, None])[..., None, None], x, torch.zeros_like(x))
    return x.unflatten(1, (blocks, BLOCK))


def _quantise(x):
    """Codes (as float) and scales of [..., 64, h, d] blocks; one scale for each block and head."""
    x = x.float()
    scale = x.abs().amax(dim=(-3, -1), keepdim=True) / 127
    c = torch.where(scale > 0, (x / scale).round().clamp(-127, 127), torch.zeros_like(x))
    return c, scale


def _plain_append(state, k, v, lens, off, n_new, blocks):
    """Puts the new tokens in place; returns the touched blocks as 16-bit values, [b, blocks * 64, h, d] each."""
    first = lens // BLOCK
    j = torch.arange(blocks, device=lens.device)
    end = lens + n_new
    full = (first[:, None] + j + 1) * BLOCK <= end[:, None]
    columns = state["table"].shape[1]
    page = state["table"].gather(1, (first[:, None] + j).clamp(max=columns - 1))
    page = torch.where(full, page, torch.full_like(page, state["k"].shape[0] - 1))  # the pool's last block is no sequence's
    left = (end % BLOCK)[:, None, None, None]
    got = []
    for kv, new in (("k", k), ("v", v)):
        x = _window(state, kv, new, lens, off, n_new, blocks)
        c, scale = _quantise(x)
        codes = c.to(torch.int8).permute(0, 1, 3, 2, 4)
        state[kv][page] = codes.transpose(-1, -2) if kv == "v" else codes
        state[kv + "_scale"][page] = scale[:, :, 0, :, 0]
        # the last touched block, if it is not complete, is the new tail
        last = (end // BLOCK - first).clamp(max=blocks - 1)
        t = x.gather(1, last[:, None, None, None, None].expand(-1, 1, *x.shape[2:]))[:, 0].permute(0, 2, 1, 3)
        keep = state[kv + "_tail"]
        t = t.transpose(2, 3) if kv == "v" else t
        place = torch.arange(BLOCK, device=lens.device).view((1, 1, 1, -1) if kv == "v" else (1, 1, -1, 1))
        keep.copy_(torch.where((place < left) & (end > lens)[:, None, None, None], t, keep))
        got.append(torch.where(full[:, :, None, None, None], (c * scale).to(x.dtype), x).flatten(1, 2))
    return got


def _held(state, kv, stored):
    """What the cache stands for, as [b, h, tokens, d] in 32 bits."""
    x = state[kv][state["table"]].float() * state[kv + "_scale"][state["table"]][..., None, None]
    tail = state[kv + "_tail"].float()
    last = (stored // BLOCK).clamp(max=x.shape[1] - 1)
    at = torch.arange(x.shape[0], device=x.device)
    x[at, last] = torch.where((stored % BLOCK > 0)[:, None, None, None], tail, x[at, last])
    x = x.transpose(-1, -2) if kv == "v" else x
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attend(state, q, lens, off, n_new, new, group, scale, causal):
    b, dev = lens.shape[0], lens.device
    stored = lens + n_new if causal else lens
    k, v = _held(state, "k", stored), _held(state, "v", stored)
    heads, d = k.shape[1], k.shape[3]
    i = torch.arange(new, device=dev)
    row = (off[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q[row].float().view(b, new, heads, group, d).permute(0, 2, 1, 3, 4).reshape(b, heads, new * group, d)
    s = torch.matmul(x, k.transpose(-1, -2).contiguous()) * scale
    s = s.view(b, heads, new, group, -1)
    seen = lens[:, None] + i + 1 if causal else lens[:, None].expand(b, new)
    hidden = torch.arange(k.shape[2], device=dev) >= seen[..., None]
    s = s.masked_fill(hidden[:, None, :, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    v = torch.where((torch.arange(v.shape[2], device=dev) < stored[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.view(b, heads, new * group, -1), v).view(b, heads, new, group, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(b, new, heads * group, d)
    r = torch.arange(q.shape[0], device=dev)
    of = torch.searchsorted(off, r, right=True) - 1
    return o[of, r - off[of]].to(q.dtype)


# ---------------------------------------------------------------------------------------------------
# what is measured
# ---------------------------------------------------------------------------------------------------
def _touched(case):
    return (case["new_hi"] + BLOCK - 2) // BLOCK + 1


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), TYPES[case["dtype"]]
    b, h, d, g = case["seqs"], case["heads"], case["dim"], case["group"]
    rng = random.Random(seed)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    new, hist = _counts(case, rng)
    most = max(case["hist_hi"] + case["new_hi"], 1)
    columns = -(-most // BLOCK)
    pages = list(range(b * columns))
    if case["paged"]:
        rng.shuffle(pages)
    total = sum(new)

    def ints(v):
        return torch.tensor(v, dtype=torch.int64).to(dev)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)

    # keys have a mean of their own in each channel, and a few channels are larger than the others
    mean, width = normal(1, h, d), 1 + 2 * (torch.rand((1, h, d), generator=gen, device=dev) > 0.95)

    def keys(n):
        return ((normal(n, h, d) + 0.5 * mean) * width).to(dtype)

    def values(n):
        return normal(n, h, d).to(dtype)

    n_blocks = b * columns + 1  # one more than the table names
    state = {
        "case": case,
        "k": torch.zeros((n_blocks, h, BLOCK, d), dtype=torch.int8, device=dev),
        "v": torch.zeros((n_blocks, h, d, BLOCK), dtype=torch.int8, device=dev),
        "k_scale": torch.zeros((n_blocks, h), device=dev),
        "v_scale": torch.zeros((n_blocks, h), device=dev),
        "k_tail": torch.zeros((b, h, BLOCK, d), dtype=dtype, device=dev),
        "v_tail": torch.zeros((b, h, d, BLOCK), dtype=dtype, device=dev),
        "table": ints(pages).view(b, columns),
    }
    # what is in the cache before the call: the history, and for causal attention alone the new tokens too
    held = [x + y for x, y in zip(hist, new)] if case["op"] == "attend" and case["causal"] else hist
    if max(held) > 0:
        ends = [0]
        for x in held:
            ends.append(ends[-1] + x)
        _plain_append(state, keys(ends[-1]), values(ends[-1]), ints([0] * b), ints(ends), ints(held), -(-max(held) // BLOCK))
    ends = [0]
    for x in new:
        ends.append(ends[-1] + x)
    lens = ints(hist)
    state |= {"new_k": keys(total), "new_v": values(total), "q": normal(total, h * g, d).to(dtype)}
    state |= {"lens64": lens, "off64": ints(ends), "new64": ints(new), "scale": 1.2 / math.sqrt(d)}
    # the same numbers as a program hands them to the framework
    state |= {"lens": lens.int(), "off": ints(ends).int(), "table32": state["table"].int(),
              "first": (lens // BLOCK * BLOCK).int(), "after": (lens + ints(new)).int(), "total": total}
    if own:
        if "open-whisper-kit_amd/python" not in sys.path:
            sys.path.insert(0, "open-whisper-kit_amd/python")
        import owk_kv8

        state["cache"] = owk_kv8.Cache.of(state["k"], state["v"], state["k_scale"], state["v_scale"], state["k_tail"],
                                          state["v_tail"], state["table32"])
    return state


def _with_state(state, out):
    """The output of a step and the state that it changed (the codes show in the output, and in the append cases)."""
    return {"out": out, "k_tail": state["k_tail"], "v_tail": state["v_tail"], "k_scale": state["k_scale"][:-1],
            "v_scale": state["v_scale"][:-1]}


def run(state):
    case = state["case"]
    new, op = case["new_hi"], case["op"]
    if own:
        cache = state["cache"]
        off = state["off"]
        if op != "attend":
            cache.append(state["new_k"], state["new_v"], state["lens"], off=off, max_new=new)
        if op == "append":
            return cache.read(state["after"], first=state["first"], max_tokens=_touched(case) * BLOCK)
        out = cache.attend(state["q"], state["lens"], off=off, max_new=new, max_len=case["hist_hi"] + new,
                           scale=state["scale"], causal=case["causal"])
        return _with_state(state, out) if op == "step" else out
    lens, off, n_new = state["lens64"], state["off64"], state["new64"]
    if op != "attend":
        got = _plain_append(state, state["new_k"], state["new_v"], lens, off, n_new, _touched(case))
        if op == "append":
            return tuple(got)
    out = _plain_attend(state, state["q"], lens, off, n_new, new, case["group"], state["scale"], case["causal"])
    return _with_state(state, out) if op == "step" else out


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits, a sequence at a time
# ---------------------------------------------------------------------------------------------------
def _stands_for(x, n):
    """What the cache stands for once it holds x [tokens, h, d]: complete blocks rounded to their codes."""
    x = x[:n].double()
    whole = n // BLOCK * BLOCK
    blocks = x[:whole].reshape(-1, BLOCK, x.shape[1], x.shape[2])
    unit = blocks.abs().amax(dim=(1, 3), keepdim=True) / 127
    codes = torch.round(blocks / unit.clamp(min=1e-300))
    return torch.cat([(codes * unit).reshape(whole, x.shape[1], x.shape[2]), x[whole:]])


def _decode(state, kv, s, n):
    """Sequence s's first n tokens as the state's codes, scales and tail say them, [n, h, d]."""
    whole = n // BLOCK
    page = state["table"][s, :whole]
    x = state[kv][page].double() * state[kv + "_scale"][page].double()[..., None, None]
    tail = state[kv + "_tail"][s].double()
    if kv == "v":
        x, tail = x.transpose(2, 3), tail.transpose(1, 2)
    x = x.transpose(1, 2).reshape(whole * BLOCK, x.shape[1], x.shape[3])
    return torch.cat([x, tail.transpose(0, 1)[: n - whole * BLOCK]])


def exact(case, seed):
    state = prepare(case, seed)
    lens, off, op = state["lens64"].tolist(), state["off64"].tolist(), case["op"]
    h, g, d = case["heads"], case["group"], case["dim"]
    window = _touched(case) * BLOCK
    outs, back = [], ([], [])
    for s in range(case["seqs"]):
        n, lo, hi = lens[s], off[s], off[s + 1]
        held = {}
        for i, kv in enumerate("kv"):
            if op == "attend":
                held[kv] = _decode(state, kv, s, n + (hi - lo if case["causal"] else 0))
                continue
            base = n // BLOCK * BLOCK  # the blocks before this one stay as they are
            old = _decode(state, kv, s, n)
            later = _stands_for(torch.cat([old[base:], state["new_" + kv][lo:hi].double()]), n - base + hi - lo)
            held[kv] = torch.cat([old[:base], later])
            if op == "append":
                pad = torch.zeros((window - later.shape[0], h, d), dtype=torch.float64, device=later.device)
                back[i].append(torch.cat([later, pad]))
        if op == "append":
            continue
        q = state["q"][lo:hi].double().view(hi - lo, h, g, d)
        o = torch.zeros((hi - lo, h, g, d), dtype=torch.float64, device=q.device)
        for head in range(h):
            logits = (q[:, head].reshape(-1, d) @ held["k"][:, head].T).view(hi - lo, g, -1) * state["scale"]
            if case["causal"]:
                place = torch.arange(logits.shape[-1], device=q.device)
                mine = n + torch.arange(hi - lo, device=q.device)
                logits[(place[None] > mine[:, None])[:, None].expand_as(logits)] = -math.inf
            if logits.shape[-1]:
                o[:, head] = torch.softmax(logits, dim=-1).reshape((hi - lo) * g, -1).matmul(held["v"][:, head]).view(hi - lo, g, d)
        outs.append(o.view(hi - lo, h * g, d))
    if op == "append":
        return torch.stack(back[0]), torch.stack(back[1])
    out = torch.cat(outs)
    return {"out": out, "k_tail": None, "v_tail": None, "k_scale": None, "v_scale": None} if op == "step" else out
