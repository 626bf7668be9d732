"""The 8-bit key/value cache (include/owk_kv8.h) against its definition in 64 bits.

Codes, scales and tails are compared bit for bit. Attention is compared element by element with a bound
that follows from the kernels' arithmetic (`_attend_bound`): f32 sums, queries in 15-bit fixed point of
their row's largest element, probabilities rounded to 14 bits of their block's largest or to half
precision, one rounding to the output's type."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import owk
import owk_kv8 as KV

gpu = pytest.mark.gpu
BLOCK = 64
F16, BF16 = torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------------------------------
# the definition, on the CPU
# ---------------------------------------------------------------------------------------------------
def quantise(x):
    """[64, d] values of one block and head -> codes (float64), scale (f32 arithmetic, as defined)."""
    x = x.float().numpy()
    with np.errstate(all="ignore"):
        top = np.float32(np.abs(x).max())
        if not np.isfinite(x).all():
            return torch.zeros(x.shape, dtype=torch.float64), float("nan")
        scale = np.float32(top / np.float32(127))
        c = np.clip(np.rint((x / scale).astype(np.float32)), -127, 127) if scale > 0 else np.zeros_like(x)
    return torch.from_numpy(c.astype(np.float64)), float(scale)


class Model:
    """What a cache should hold: the tokens of each sequence as given, in 16 bits."""

    def __init__(self, n_seqs, heads, dim, dtype):
        self.heads, self.dim, self.dtype = heads, dim, dtype
        self.k = [torch.zeros((0, heads, dim), dtype=dtype) for _ in range(n_seqs)]
        self.v = [torch.zeros((0, heads, dim), dtype=dtype) for _ in range(n_seqs)]

    def append(self, s, start, k, v):
        self.k[s] = torch.cat([self.k[s][:start], k.cpu()])
        self.v[s] = torch.cat([self.v[s][:start], v.cpu()])

    def held(self, s, kv):
        """float64 [tokens, heads, dim]: complete blocks as their codes say, the rest as given."""
        x = self.k[s] if kv == "k" else self.v[s]
        out = x.double()
        for lo in range(0, x.shape[0] // BLOCK * BLOCK, BLOCK):
            for h in range(self.heads):
                c, scale = quantise(x[lo:lo + BLOCK, h])
                out[lo:lo + BLOCK, h] = c * scale
        return out


def attend(q, k, v, scale, seen, dtype):
    """q [n, hq, d], k / v float64 [tokens, h, d], seen [n] -> (out float64, bound)."""
    n, hq, d = q.shape
    g = hq // k.shape[1] if k.shape[0] else 1
    out, bound = torch.zeros((n, hq, d), dtype=torch.float64), torch.zeros((n, hq, d), dtype=torch.float64)
    half = (torch.finfo(dtype).eps / 2) if dtype != torch.float32 else 2.0 ** -24
    for i in range(n):
        if seen[i] == 0:
            continue
        for h in range(hq):
            kk, vv, x = k[:seen[i], h // g], v[:seen[i], h // g], q[i, h].double()
            s = scale * (kk @ x)
            p = torch.exp(s - s.max())
            o = (p @ vv) / p.sum()
            out[i, h] = o
            bound[i, h] = _attend_bound(x, kk, vv, scale, s, p, o, half, torch.finfo(dtype).tiny)
    return out, bound


def _attend_bound(q, k, v, scale, s, p, o, half, tiny):
    # a score: queries off by 2^-15 of the row's largest element (fixed point) or 2^-11 of a step of it below the
    # normal range (half precision, scaled), keys exact; then a handful of f32 roundings of values up to max|s|
    ds = abs(scale) * q.abs().max() * 2.0 ** -15 * k.abs().sum(1) + 8 * 2.0 ** -24 * (s.abs().max() + s.abs()) + 2.0 ** -22
    # a probability: its score's error, 2^-11 of itself (half precision) and 2^-15 of its block's largest (fixed point)
    blocks = torch.arange(p.shape[0]) // BLOCK
    top = torch.zeros(int(blocks[-1]) + 1, dtype=p.dtype).scatter_reduce(0, blocks, p, "amax")[blocks]
    dp = p * (torch.expm1(ds) + 2.0 ** -11) + top * 2.0 ** -15
    # the quotient moves by sum dp_j |v_j - o| / sum p; f32 sums of n terms by n steps at most
    first = (dp[:, None] * (v - o).abs()).sum(0) / p.sum()
    sums = (p.shape[0] + 16) * 2.0 ** -24 * (p[:, None] * v.abs()).sum(0) / p.sum()
    return 1.05 * (first + sums) + half * o.abs() + tiny


def pages(n_seqs, blocks, seed, spare=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n_seqs * blocks + spare, generator=g)[: n_seqs * blocks].view(n_seqs, blocks).int()


def make(n_seqs, heads, dim, tokens, dtype, paged=False, seed=0):
    blocks = -(-max(tokens, 1) // BLOCK)
    table = pages(n_seqs, blocks, seed).cuda() if paged else None
    return KV.Cache(n_seqs, heads, dim, tokens, dtype, "cuda", n_blocks=n_seqs * blocks + 3, table=table)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def normal(gen, *shape, dtype, width=1.0):
    return (torch.randn(shape, generator=gen) * width).to(dtype)


def fill(cache, model, counts, seed=1, width=1.0):
    """Each sequence gets counts[s] tokens in one joined call."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(counts)
    k, v = (normal(gen, total, cache.n_heads, cache.head_dim, dtype=cache.dtype, width=width) for _ in "kv")
    off = np.concatenate([[0], np.cumsum(counts)]).tolist()
    cache.append(k.cuda(), v.cuda(), ints([0] * len(counts)), off=ints(off), max_new=max(max(counts), 1))
    for s in range(len(counts)):
        model.append(s, 0, k[off[s]:off[s + 1]], v[off[s]:off[s + 1]])


def assert_held(cache, model, lens):
    n = max(max(lens), 1) + 5
    k, v = cache.read(ints(lens), n)
    for s, x in enumerate(lens):
        for kv, got in (("k", k[s].cpu()), ("v", v[s].cpu())):
            want = model.held(s, kv)
            # a code times its scale, rounded once to f32 and once to the type
            want = want.float().to(cache.dtype)
            torch.testing.assert_close(got[:x], want, rtol=0, atol=0, equal_nan=True, msg=f"sequence {s} {kv}")
            assert not got[x:].any()


def check_attend(cache, model, lens, new, group, causal, *args, **kw):
    """Query rows new[b] for each sequence b; lens: tokens before the call's own. More than 32 rows a head can run in either
    form, by how much work there is: both are checked, whichever this call would get."""
    L = KV.load()
    for rows in (32, 1 << 30) if max(new) * group > 32 else (0,):
        cache._ws.clear()  # sizes of the other form's workspaces
        L.owk_debug_kv8_set_many_rows(rows)
        try:
            _check_attend(cache, model, lens, new, group, causal, *args, **kw)
        finally:
            L.owk_debug_kv8_set_many_rows(0)
            cache._ws.clear()


def _check_attend(cache, model, lens, new, group, causal, layout="joined", out_type=None, scale=None, seed=3, width=1.0, max_len=0,
                  rows=None):
    gen = torch.Generator().manual_seed(seed)
    hq, d, n = cache.n_heads * group, cache.head_dim, len(lens)
    scale = d ** -0.5 if scale is None else scale
    rows = rows or [normal(gen, x, hq, d, dtype=cache.dtype, width=width) for x in new]
    out_type = out_type or cache.dtype
    mark = 7.25
    if layout == "joined":
        off = np.concatenate([[0], np.cumsum(new)]).tolist()
        q = torch.cat(rows + [normal(gen, 2, hq, d, dtype=cache.dtype)]).cuda()  # two rows behind the last entry's
        out = torch.full((q.shape[0], hq, d), mark, dtype=out_type, device="cuda")
        got = cache.attend(q, ints(lens), off=ints(off), max_new=max(new), max_len=max_len, scale=scale, causal=causal, out=out)
        mine = [got[off[b]:off[b + 1]] for b in range(n)]
        rest = [got[off[-1]:]]
    else:
        most = max(new) + 1
        q = torch.zeros((n, most, hq, d), dtype=cache.dtype)
        for b in range(n):
            q[b, :new[b]] = rows[b]
        q = q.cuda()
        out = torch.full(q.shape, mark, dtype=out_type, device="cuda")
        if layout == "strided":  # heads outermost, odd row strides, an unaligned base
            store = torch.zeros((n, hq, most, d + 3), dtype=cache.dtype, device="cuda")
            q = store[..., 1:d + 1].permute(0, 2, 1, 3).copy_(q)
            out = torch.full((n, hq, most, d + 5), mark, dtype=out_type, device="cuda")[..., 3:d + 3].permute(0, 2, 1, 3)
        got = cache.attend(q, ints(lens), count=ints(new), max_len=max_len, scale=scale, causal=causal, out=out)
        mine = [got[b, :new[b]] for b in range(n)]
        rest = [got[b, new[b]:] for b in range(n)]
    assert got.data_ptr() == out.data_ptr()
    for x in rest:
        assert (x == mark).all(), "rows that are no entry's were written"
    for b in range(n):
        seen = [lens[b] + i + 1 if causal else lens[b] for i in range(new[b])]
        want, bound = attend(rows[b], model.held(b, "k"), model.held(b, "v"), scale, seen, out_type)
        x = mine[b].cpu().double()
        assert x.shape == want.shape
        nan = want.isnan()
        assert torch.equal(x.isnan(), nan), f"entry {b}"
        err = ((x - want).abs() - bound).nan_to_num(nan=-1.0)
        at = int(err.argmax()) if err.numel() else 0
        assert err.numel() == 0 or err.max() <= 0, (
            f"entry {b} ({lens[b]} tokens) element {np.unravel_index(at, tuple(want.shape))}: {x.flatten()[at]:.6g}, "
            f"wanted {want.flatten()[at]:.6g} +- {bound.flatten()[at]:.3g}")


# ---------------------------------------------------------------------------------------------------
# CPU: refusals and bounds
# ---------------------------------------------------------------------------------------------------
class Raw:
    """The C entries with structures passed by address (the binding itself passes packed bytes)."""

    def __getattr__(self, name):
        def call(*args):
            return getattr(KV.load(), name)(*[C.addressof(a) if isinstance(a, C.Structure) else a for a in args])

        return call


def _desc(**kw):
    d = dict(device=0, dtype=0, head_dim=64, n_heads=2, n_seqs=3, n_blocks=12, max_blocks=4, k=4096, v=8192, k_scale=4096,
             v_scale=4096, k_tail=4096, v_tail=4096, table=None)
    d.update(kw)
    return KV.CacheDesc(*[d[f[0]] for f in KV.CacheDesc._fields_])


def _batch(**kw):
    d = dict(n=2, max_new=5, rows=10, lens=4096, seq=None, off=None, count=None)
    d.update(kw)
    return KV.Batch(*[d[f[0]] for f in KV.Batch._fields_])


def _rows(data=4096, entry=0, row=128, head=64):
    return KV.Rows(data, entry, row, head)


def _params(**kw):
    d = dict(n_q_heads=4, causal=0, out_type=0, max_len=0, scale=0.125)
    d.update(kw)
    return KV.AttendParams(*[d[f[0]] for f in KV.AttendParams._fields_])


BAD_CACHE = [dict(dtype=2), dict(dtype=-1), dict(head_dim=0), dict(head_dim=80), dict(head_dim=256), dict(n_heads=0),
             dict(n_heads=40000), dict(n_seqs=0), dict(n_blocks=0), dict(max_blocks=0), dict(max_blocks=1 << 25), dict(k=None),
             dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k_tail=None), dict(v_tail=None), dict(k=4100),
             dict(v_tail=4104), dict(k_scale=4104), dict(table=4097), dict(n_blocks=11)]
BAD_BATCH = [dict(n=-1), dict(n=70000), dict(max_new=-1), dict(max_new=1 << 23), dict(lens=None), dict(lens=4098),
             dict(off=4096, rows=-1), dict(seq=4097), dict(off=4097), dict(count=4099)]
BAD_ROWS = [dict(data=None), dict(data=4097), dict(row=-1), dict(head=-64), dict(entry=-5), dict(row=1 << 41)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_refused_caches(bad):
    L = Raw()
    d = _desc(**bad)
    assert L.owk_kv8_append(d, _batch(), _rows(), _rows(), None) == -1
    assert L.owk_kv8_error()
    assert L.owk_kv8_attend(d, _batch(), _params(), _rows(), _rows(), None, 0, None) == -1
    assert L.owk_kv8_attend_workspace(d, _batch(), _params()) == 0
    assert L.owk_kv8_read(d, 2, 5, 4096, None, None, _rows(), _rows(), None) == -1


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_refused_batches(bad):
    L = Raw()
    d, b = _desc(), _batch(**bad)
    assert L.owk_kv8_append(d, b, _rows(), _rows(), None) == -1
    assert L.owk_kv8_attend(d, b, _params(), _rows(), _rows(), None, 0, None) == -1
    assert L.owk_kv8_attend_workspace(d, b, _params()) == 0


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_refused_tensors(bad):
    L = Raw()
    d, r = _desc(), _rows(**bad)
    assert L.owk_kv8_append(d, _batch(), r, _rows(), None) == -1
    assert L.owk_kv8_append(d, _batch(), _rows(), r, None) == -1
    assert L.owk_kv8_attend(d, _batch(), _params(), r, _rows(), None, 0, None) == -1
    assert L.owk_kv8_attend(d, _batch(), _params(), _rows(), r, None, 0, None) == -1
    assert L.owk_kv8_read(d, 2, 5, 4096, None, None, r, _rows(), None) == -1


@pytest.mark.parametrize("bad", [dict(n_q_heads=0), dict(n_q_heads=3), dict(out_type=1), dict(out_type=3), dict(max_len=-1),
                                 dict(scale=math.inf), dict(scale=math.nan)], ids=str)
def test_refused_params(bad):
    L = Raw()
    assert L.owk_kv8_attend(_desc(), _batch(), _params(**bad), _rows(), _rows(), None, 0, None) == -1
    assert L.owk_kv8_attend_workspace(_desc(), _batch(), _params(**bad)) == 0


def test_refused_workspaces():
    L = Raw()
    d, b = (_desc(n_seqs=1, n_heads=1, n_blocks=1 << 14, max_blocks=1 << 14)), _batch(n=1, max_new=1)
    need = L.owk_kv8_attend_workspace(d, b, _params(n_q_heads=1))
    if need:  # one long sequence is cut into parts
        for ws, n in ((None, 0), (4096, need - 1), (4104, need)):
            assert L.owk_kv8_attend(d, b, _params(n_q_heads=1), _rows(), _rows(), ws, n, None) == -1


@pytest.mark.parametrize("desc,batch,params", [
    (dict(), dict(max_new=1 << 22), dict(n_q_heads=4)),                               # rows of a head
    (dict(), dict(max_new=1 << 20), dict(n_q_heads=40000)),
    (dict(n_heads=32000), dict(n=65535, max_new=1), dict(n_q_heads=32000)),           # tiles
    (dict(n_heads=32000), dict(n=2000, max_new=1), dict(n_q_heads=32000)),
    (dict(n_heads=2, n_seqs=1, n_blocks=1 << 24, max_blocks=1 << 24), dict(n=64, max_new=1), {}),  # parts of long sequences
    (dict(n_heads=2, n_seqs=1, n_blocks=1 << 24, max_blocks=1 << 24), dict(n=65535, max_new=1 << 20), {}),
])
def test_refused_sizes(desc, batch, params):
    """More workgroups than a launch can have."""
    L = Raw()
    d, b, p = _desc(**{"n_blocks": 1 << 20, **desc}), _batch(**batch), _params(**params)
    assert L.owk_kv8_attend(d, b, p, _rows(), _rows(), 4096, 1 << 62, None) == -1
    assert b"too much for one call" in KV.load().owk_kv8_error()
    assert L.owk_kv8_attend_workspace(d, b, p) == 0


def test_nothing_to_do_is_no_call():
    """Empty calls succeed without a device."""
    L = Raw()
    d = _desc()
    for b in (_batch(n=0, lens=None), _batch(max_new=0), _batch(off=4096, rows=0)):
        assert L.owk_kv8_append(d, b, _rows(), _rows(), None) == 0
        assert L.owk_kv8_attend(d, b, _params(), _rows(), _rows(), None, 0, None) == 0
    assert L.owk_kv8_read(d, 0, 5, None, None, None, _rows(), _rows(), None) == 0


def test_missing_pointers_are_refused():
    L = Raw()
    assert L.owk_kv8_append(None, _batch(), _rows(), _rows(), None) == -1
    assert L.owk_kv8_append(_desc(), None, _rows(), _rows(), None) == -1
    assert L.owk_kv8_append(_desc(), _batch(), None, _rows(), None) == -1
    assert L.owk_kv8_attend(_desc(), _batch(), None, _rows(), _rows(), None, 0, None) == -1


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        KV.Cache(1, 1, 64, 64, device="cpu")


def _host(x):
    a = np.ascontiguousarray(x, dtype=np.int32)
    return a, a.ctypes.data


def test_entries_are_bounded():
    """What the device reads from index arrays never leads out of a tensor (the kernels' own function, on the host)."""
    L = KV.load()
    L.owk_debug_kv8_entry.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.POINTER(C.c_int64)]
    big = 2 ** 31 - 1
    d = _desc()  # 3 sequences of 256 tokens
    out = (C.c_int64 * 4)()

    def entry(b, **kw):
        keep = {k: _host(v) for k, v in kw.items() if k in ("lens", "seq", "off", "count")}
        args = {k: v for k, v in kw.items() if k not in keep} | {k: v[1] for k, v in keep.items()}
        bt = _batch(**args)
        L.owk_debug_kv8_entry(C.addressof(d), C.addressof(bt), b, out)
        return list(out)

    assert entry(1, lens=[3, 70]) == [1, 70, 5, 0]
    assert entry(0, lens=[-4, 0])[1] == 0
    assert entry(0, lens=[big, 0])[1] == 256
    for s in (-1, 3, big, -big):
        assert entry(0, lens=[1, 1], seq=[s, 0])[0] == -1
    assert entry(0, lens=[1, 1], seq=[2, 2])[0] == 2
    assert entry(0, lens=[1, 1], count=[2, 9])[2] == 2
    assert entry(1, lens=[1, 1], count=[2, 9])[2] == 5  # max_new
    assert entry(1, lens=[1, 1], count=[2, -9])[2] == 0
    for off, want in (([0, 4, 9], (5, 4)), ([0, 8, 99], (2, 8)), ([0, 12, 99], (0, None)), ([0, 4, 2], (0, None)),
                      ([0, -3, 2], (0, None)), ([0, 1, big], (5, 1)), ([0, 10, 10], (0, None))):
        got = entry(1, lens=[1, 1], off=off, rows=10)
        assert got[2] == want[0] and (want[1] is None or got[3] == want[1])
        assert got[2] == 0 or (got[3] >= 0 and got[3] + got[2] <= 10)


def test_table_entries_are_bounded():
    L = KV.load()
    L.owk_debug_kv8_page.argtypes = [C.c_void_p, C.c_int, C.c_int]
    L.owk_debug_kv8_page.restype = C.c_int64
    big = 2 ** 31 - 1
    t, p = _host([[3, -1, 12, 11], [big, -big, 0, 1], [2, 2, 2, 2]])
    d = _desc(table=p)
    got = [[L.owk_debug_kv8_page(C.addressof(d), s, i) for i in range(-1, 6)] for s in range(-1, 3)]
    assert got[0] == [-1] * 7
    assert got[1] == [-1, 3, -1, -1, 11, -1, -1]
    assert got[2] == [-1, -1, -1, 0, 1, -1, -1]
    d = _desc()
    assert [L.owk_debug_kv8_page(C.addressof(d), s, i) for s, i in ((0, 0), (2, 3), (2, 4), (1, -1))] == [0, 11, -1, -1]


# ---------------------------------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------------------------------
SHAPES = [(64, F16), (128, F16), (64, BF16), (128, BF16)]


@gpu
@pytest.mark.parametrize("dim,dtype", SHAPES)
@pytest.mark.parametrize("paged", [False, True])
def test_append_and_read(dim, dtype, paged):
    lens = [0, 1, 63, 64, 65, 127, 128, 200]
    cache, model = make(len(lens), 3, dim, 256, dtype, paged), Model(len(lens), 3, dim, dtype)
    fill(cache, model, lens)
    assert_held(cache, model, lens)


@gpu
@pytest.mark.parametrize("dim,dtype", SHAPES[:1] + SHAPES[3:])
def test_codes_do_not_depend_on_the_calls(dim, dtype):
    """The same tokens in one call, one at a time and in ragged pieces: the same cache, bit for bit."""
    gen = torch.Generator().manual_seed(5)
    n, h = 2 * BLOCK + 9, 2
    k, v = (normal(gen, n, h, dim, dtype=dtype).cuda() for _ in "kv")
    caches = []
    for cuts in ([n], [1] * n, [60, 70, 1, n - 131], [64, 64, 9], [63, 2, 63, 9]):
        c = make(1, h, dim, 192, dtype)
        at = 0
        for x in cuts:
            c.append(k[None, at:at + x], v[None, at:at + x], ints([at]))
            at += x
        caches.append(c)
    for c in caches[1:]:
        for name in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(c, name), getattr(caches[0], name)), name
        assert torch.equal(c.k_tail[:, :, :9], caches[0].k_tail[:, :, :9])
        assert torch.equal(c.v_tail[..., :9], caches[0].v_tail[..., :9])


@gpu
def test_append_again_from_a_block_border():
    """Tokens from an earlier multiple of 64 on are dropped and stored anew."""
    cache, model = make(1, 2, 64, 256, F16), Model(1, 2, 64, F16)
    fill(cache, model, [150])
    gen = torch.Generator().manual_seed(9)
    k, v = (normal(gen, 40, 2, 64, dtype=F16) for _ in "kv")
    cache.append(k[None].cuda(), v[None].cuda(), ints([64]))
    model.append(0, 64, k, v)
    assert_held(cache, model, [104])
    check_attend(cache, model, [104], [3], 1, False)


@gpu
def test_append_of_some_sequences():
    """seq picks and orders sequences; counts may be zero; the others stay as they are."""
    cache, model = make(5, 2, 64, 192, F16), Model(5, 2, 64, F16)
    lens = [10, 64, 0, 130, 63]
    fill(cache, model, lens)
    gen = torch.Generator().manual_seed(2)
    k, v = (normal(gen, 3, 70, 2, 64, dtype=F16) for _ in "kv")
    pick, count = [4, 0, 3], [2, 70, 0]
    cache.append(k.cuda(), v.cuda(), ints([lens[s] for s in pick]), seq=ints(pick), count=ints(count))
    for b, s in enumerate(pick):
        model.append(s, lens[s], k[b, :count[b]], v[b, :count[b]])
        lens[s] += count[b]
    assert_held(cache, model, lens)
    kk, vv = cache.read(ints([lens[s] for s in pick]), 100, seq=ints(pick), first=ints([0, 50, 131]))
    for b, (s, first) in enumerate(zip(pick, [0, 50, 131])):
        want = model.held(s, "k").float().half()[first:first + 100]
        assert torch.equal(kk[b, :want.shape[0]].cpu(), want) and not kk[b, want.shape[0]:].any()


@gpu
@pytest.mark.parametrize("strides", ["heads first", "odd", "expanded"])
def test_append_strides(strides):
    gen = torch.Generator().manual_seed(4)
    n, h, d = 70, 3, 64
    base = normal(gen, 2, n, h, d, dtype=BF16).cuda()
    if strides == "heads first":
        x = base.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    elif strides == "odd":
        x = torch.zeros((2, n, h, d + 1), dtype=BF16, device="cuda")[..., 1:].copy_(base)
    else:
        base = base[:, :1].expand(2, n, h, d)
        x = base
    cache, model = make(2, h, d, 128, BF16), Model(2, h, d, BF16)
    cache.append(x, x, ints([0, 0]))
    for s in range(2):
        model.append(s, 0, base[s].cpu(), base[s].cpu())
    assert_held(cache, model, [n, n])


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_at_the_edges(dtype):
    """All zeros, ties between codes, the type's largest and smallest values, and values that are not finite."""
    h, d = 6, 64
    x = torch.zeros((BLOCK, h, d), dtype=dtype)
    x[3, 1, 5] = 127.0  # scale 1: halves are ties
    x[:, 1, :32] = (torch.arange(BLOCK)[:, None] + torch.arange(32) / 2 - 40).to(dtype)
    x[3, 1, 5] = 127.0
    x[:, 2] = torch.finfo(dtype).max * torch.linspace(-1, 1, BLOCK)[:, None].to(dtype)
    x[:, 3] = torch.finfo(dtype).smallest_normal * torch.linspace(0, 0.02, BLOCK)[:, None].to(dtype)
    x[7, 4, 9] = math.inf
    x[9, 5, 0] = math.nan
    cache, model = make(1, h, d, 128, dtype), Model(1, h, d, dtype)
    cache.append(x[None].cuda(), x.flip(0)[None].cuda(), ints([0]))
    model.append(0, 0, x, x.flip(0))
    k, v = (t.cpu() for t in cache.read(ints([64]), 64))
    for got, kv in ((k, "k"), (v, "v")):
        want = model.held(0, kv).float().to(dtype)
        torch.testing.assert_close(got[0], want, rtol=0, atol=0, equal_nan=True)
    assert k[0, :, 4:].isnan().all() and not k[0, :, :4].isnan().any()


LENS = [0, 1, 2, 31, 63, 64, 65, 100, 127, 128, 300, 449]


@gpu
@pytest.mark.parametrize("dim,dtype", SHAPES)
@pytest.mark.parametrize("layout", ["joined", "padded", "strided"])
def test_cross_rows(dim, dtype, layout):
    """Every row sees the whole sequence; none, one or several rows each."""
    cache, model = make(len(LENS), 2, dim, 450, dtype, paged=layout != "padded"), Model(len(LENS), 2, dim, dtype)
    fill(cache, model, LENS)
    check_attend(cache, model, LENS, [1 + (s % 3) for s in range(len(LENS))], 1, False, layout)
    check_attend(cache, model, LENS, [0 if s % 2 else 2 for s in range(len(LENS))], 3, False, layout)


@gpu
@pytest.mark.parametrize("dim,dtype", SHAPES)
@pytest.mark.parametrize("group", [1, 2, 5, 8])
def test_one_causal_token(dim, dtype, group):
    cache, model = make(len(LENS), 2, dim, 450, dtype, paged=True), Model(len(LENS), 2, dim, dtype)
    fill(cache, model, [x + 1 for x in LENS])
    check_attend(cache, model, LENS, [1] * len(LENS), group, True)


@gpu
@pytest.mark.parametrize("dim,dtype", SHAPES)
@pytest.mark.parametrize("new", [2, 16, 17, 33, 64, 130])
def test_causal_chunk(dim, dtype, new):
    lens = [0, 1, 50, 64, 127, 200]
    counts = [new, max(new - 1, 1), new, 1, new, new]
    cache, model = make(len(lens), 2, dim, 400, dtype, paged=True), Model(len(lens), 2, dim, dtype)
    fill(cache, model, [x + n for x, n in zip(lens, counts)])
    check_attend(cache, model, lens, counts, 2 if new < 64 else 1, True)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [40, 100, 257])
def test_cross_prompt(dtype, new):
    lens = [150, 64, 0, 29]
    cache, model = make(4, 2, 64, 192, dtype), Model(4, 2, 64, dtype)
    fill(cache, model, lens)
    check_attend(cache, model, lens, [new, new // 2, 3, new - 1], 1, False)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_float_outputs(dim, dtype):
    cache, model = make(3, 2, dim, 300, dtype), Model(3, 2, dim, dtype)
    fill(cache, model, [257, 64, 0])
    check_attend(cache, model, [257, 64, 0], [1, 2, 1], 1, False, out_type=torch.float32)
    check_attend(cache, model, [257, 64, 0], [70, 33, 64], 1, False, out_type=torch.float32)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_large_scores(dim, dtype):
    """One key far ahead of the rest, and widely spread scores."""
    cache, model = make(2, 2, dim, 400, dtype), Model(2, 2, dim, dtype)
    fill(cache, model, [333, 70], width=4.0)
    check_attend(cache, model, [333, 70], [2, 1], 1, False, width=4.0, scale=0.2)
    check_attend(cache, model, [333, 70], [64, 40], 1, False, width=4.0, scale=0.2)
    check_attend(cache, model, [333, 70], [2, 1], 1, False, width=4.0, scale=-0.2)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("new", [2, 70])
def test_blocks_of_different_size(dim, dtype, new):
    """Values of a block 2^19 (bf16: up to 2^100) apart from the next one's, and rows that see little of the large ones:
    what the small ones add keeps its bits."""
    powers = [9, -10, -9, 0, -10, 3, 9, -12, -10] if dtype == F16 else [60, -20, -40, 3, -40, 40, 60, -30, -40]
    n = 64 * len(powers) + 5
    cache, model = make(1, 2, dim, n, dtype), Model(1, 2, dim, dtype)
    gen = torch.Generator().manual_seed(12)
    k, v = normal(gen, n, 2, dim, dtype=dtype, width=0.3), normal(gen, n, 2, dim, dtype=dtype)
    size = torch.tensor(powers + powers[:1]).repeat_interleave(64)[:n, None, None].double()
    v = (v.double() * 2.0 ** size).to(dtype)
    k[:, :, 0] = torch.where(size[:, :, 0] > -9, -5.0, 5.0).to(dtype)  # the large ones: scores 100 below
    cache.append(k[None].cuda(), v[None].cuda(), ints([0]))
    model.append(0, 0, k, v)
    q = normal(gen, new, 2, dim, dtype=dtype, width=0.3)
    q[:, :, 0] = 10.0
    q[1::2, :, 0] = 0.0  # every other row sees all of them alike
    check_attend(cache, model, [n], [new], 1, False, rows=[q], scale=1.0)
    check_attend(cache, model, [n - new], [new], 1, True, rows=[q], scale=1.0, out_type=torch.float32)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("new", [3, 20, 100])
def test_joined_parts(dim, dtype, new):
    """A few parts of the keys, for few rows and for many: joined a row at a time."""
    lens, counts = [2500, 600, 2111, 64], [new, 1, new, new - 1]
    held = [x + n for x, n in zip(lens, counts)]
    cache, model = make(4, 1, dim, 2624, dtype, paged=True), Model(4, 1, dim, dtype)
    fill(cache, model, held)
    check_attend(cache, model, lens, counts, 1, True, layout="strided")
    check_attend(cache, model, held, [1, new, 0, new], 2, False, out_type=torch.float32)


@gpu
@pytest.mark.parametrize("max_len", [1, 64, 700, 100000])
@pytest.mark.parametrize("new", [1, 40])
def test_lengths_beyond_the_hint(max_len, new):
    """max_len only decides how the work is cut: sequences that hold more, or far less, come out right."""
    lens = [1500, 0, 700, 63]
    cache, model = make(4, 2, 64, 1600, F16), Model(4, 2, 64, F16)
    fill(cache, model, lens)
    check_attend(cache, model, lens, [new] * 4, 1, False, max_len=max_len)


@gpu
def test_entries_that_share_a_sequence():
    """One sequence named by several entries of an attend call, at different lengths."""
    cache, model = make(2, 2, 64, 400, F16), Model(2, 2, 64, F16)
    fill(cache, model, [321, 130])
    gen = torch.Generator().manual_seed(14)
    seq, lens, new = [0, 1, 0, 0], [321, 130, 320 - 320 % 64, 64], 3
    q = normal(gen, 4, new, 4, 64, dtype=F16)
    got = cache.attend(q.cuda(), ints(lens), seq=ints(seq)).cpu().double()
    for b in range(4):
        want, bound = attend(q[b], model.held(seq[b], "k"), model.held(seq[b], "v"), 0.125, [lens[b]] * new, F16)
        assert ((got[b] - want).abs() <= bound).all(), b


@gpu
@pytest.mark.parametrize("new", [1, 40])
def test_output_over_the_queries(new):
    """A call may write where its queries are."""
    cache, model = make(2, 2, 64, 200, F16), Model(2, 2, 64, F16)
    fill(cache, model, [190, 65])
    gen = torch.Generator().manual_seed(15)
    q = normal(gen, 2, new, 4, 64, dtype=F16).cuda()
    want = cache.attend(q, ints([190, 65]))
    assert torch.equal(cache.attend(q, ints([190, 65]), out=q), want)


@gpu
@pytest.mark.parametrize("new", [1, 48])
def test_long_cache(new):
    """Work cut along the keys and joined; positions of the last tokens."""
    cache, model = make(2, 1, 64, 9000, F16, paged=True), Model(2, 1, 64, F16)
    fill(cache, model, [8999, 4097])
    check_attend(cache, model, [8999, 4097], [new, 1], 1, False)
    check_attend(cache, model, [8999 - new, 4096], [new, 1], 1, True)


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_poisoned_tokens(causal, new):
    """What is not finite shows where it is seen and nowhere else: a block in all rows that see any of it, a
    tail token in the rows that see it; memory behind the last token is never looked at."""
    dim, dtype, lens = 64, F16, [160, 160, 160, 130]
    counts = [x + (new if causal else 0) for x in lens]
    cache, model = make(4, 1, dim, 256, dtype), Model(4, 1, dim, dtype)
    cache.k_tail.fill_(math.nan)
    cache.v_tail.fill_(math.inf)
    cache.k_scale.fill_(math.nan)
    cache.v_scale.fill_(math.nan)
    fill(cache, model, counts)
    check_attend(cache, model, lens, [new] * 4, 1, causal)
    # a value in the tail of sequence 1, its last token
    at = counts[1] - 1
    if at % BLOCK != BLOCK - 1 and at // BLOCK == counts[1] // BLOCK:
        cache.v_tail[1, 0, 5, at % BLOCK] = math.inf
        gen = torch.Generator().manual_seed(3)
        q = normal(gen, 4, new, 1, dim, dtype=dtype).cuda()
        clean = cache.attend(q, ints(lens), causal=causal)
        sees = [lens[1] + i + 1 > at if causal else True for i in range(new)]
        for i in range(new):
            row = clean[1, i, 0]
            assert not row[5].isfinite() if sees[i] else row.isfinite().all(), i
        assert clean[0].isfinite().all() and clean[2].isfinite().all() and clean[3].isfinite().all()


@gpu
def test_hidden_pages_and_bad_sequences():
    """A block whose table entry is out of the pool stores nothing and has no keys; an entry without a sequence gets zeros."""
    cache, model = make(3, 2, 64, 256, F16, paged=True), Model(3, 2, 64, F16)
    lens = [200, 140, 70]
    fill(cache, model, lens)
    good = cache.table.clone()
    before = cache.k.clone()
    for bad in (-1, 10 ** 9, cache.k.shape[0]):
        cache.table.copy_(good)
        cache.table[0, 1] = bad
        gen = torch.Generator().manual_seed(1)
        q = normal(gen, 3, 2, 2, 64, dtype=F16)
        out = cache.attend(q.cuda(), ints(lens), seq=ints([0, 7, 2])).cpu().double()
        k, v = model.held(0, "k"), model.held(0, "v")
        keep = torch.cat([torch.arange(0, 64), torch.arange(128, 200)])
        want, bound = attend(q[0], k[keep], v[keep], 0.125, [keep.numel()] * 2, F16)
        # the bound's blocks of 64 start elsewhere than the cache's: twice is ample for the rounding of probabilities
        assert ((out[0] - want).abs() <= 2 * bound).all()
        assert not out[1].any()
        rk, _ = cache.read(ints(lens), 200)
        assert not rk[0, 64:128].any() and torch.equal(rk[0, :64].cpu(), k[:64].float().half())
        x = torch.ones((1, 128, 2, 64), dtype=F16, device="cuda")
        cache.append(x, x, ints([0]), seq=ints([-1]))
        assert torch.equal(cache.k, before)
        cache.append(x[:, :64], x[:, :64], ints([64]), seq=ints([0]))
        assert torch.equal(cache.k, before)


@gpu
def test_append_beyond_the_capacity_is_cut():
    cache, model = make(2, 1, 64, 128, F16), Model(2, 1, 64, F16)
    gen = torch.Generator().manual_seed(1)
    k = normal(gen, 2, 150, 1, 64, dtype=F16)
    cache.append(k.cuda(), k.cuda(), ints([0, 100]))
    got, _ = cache.read(ints([128, 100]), 128)
    model.append(0, 0, k[0, :128], k[0, :128])
    assert torch.equal(got[0].cpu(), model.held(0, "k").float().half())
    assert not cache.k[4:].any()  # the pool behind the two sequences


@gpu
def test_decoding_run():
    """Prompt chunks, then tokens one by one, ragged over the sequences, two layers sharing lens: every output of the run."""
    n, h, g, d, dtype = 4, 2, 2, 64, F16
    caches = [make(n, h, d, 256, dtype, paged=True, seed=s) for s in range(2)]
    models = [Model(n, h, d, dtype) for _ in range(2)]
    gen = torch.Generator().manual_seed(8)
    lens = ints([0] * n)
    at = [0] * n
    for step, counts in enumerate([[20, 64, 1, 0], [50, 3, 70, 62]] + [[1, 1, 1, 1]] * 6 + [[1, 0, 2, 1], [5, 61, 1, 30]]):
        most = max(counts)
        for cache, model in zip(caches, models):
            k, v = (normal(gen, n, most, h, d, dtype=dtype) for _ in "kv")
            cache.append(k.cuda(), v.cuda(), lens, count=ints(counts))
            for s in range(n):
                model.append(s, at[s], k[s, :counts[s]], v[s, :counts[s]])
            check_attend(cache, model, at, counts, g, True, layout="padded" if step % 2 else "joined", seed=step)
        lens += ints(counts)
        at = [a + c for a, c in zip(at, counts)]
    for cache, model in zip(caches, models):
        assert_held(cache, model, at)


@gpu
@pytest.mark.parametrize("long", [False, True])
def test_captured_step(long):
    """A step captured once and replayed with lengths, tokens and queries that move on: each replay equals the eager
    call; two graphs hold workspaces of their own."""
    n, h, d, cap = (1, 1, 64, 6000) if long else (3, 2, 64, 512)
    start = [5500] if long else [62, 0, 126]
    eager, graphed = make(n, h, d, cap, F16), make(n, h, d, cap, F16)
    gen = torch.Generator().manual_seed(1)
    k0, v0 = (normal(gen, sum(start), h, d, dtype=F16).cuda() for _ in "kv")
    off = ints(np.concatenate([[0], np.cumsum(start)]).tolist())
    for c in (eager, graphed):
        c.append(k0, v0, ints([0] * n), off=off, max_new=max(start))
    k, v, q = (torch.zeros((n, 1, h, d), dtype=F16, device="cuda") for _ in "kvq")
    lens = ints(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                graphed.append(k, v, lens)
                outs.append(graphed.attend(q, lens, causal=True))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(5):
        for x in (k, v, q):
            x.copy_(normal(gen, n, 1, h, d, dtype=F16))
        eager.append(k, v, lens)
        want = eager.attend(q, lens, causal=True)
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[step % 2], want), step
        other = eager.attend(q, lens, causal=False)  # eager work between the replays
        assert other.isfinite().all()
        lens += 1


@gpu
@pytest.mark.parametrize("many", [32, 1 << 30])
def test_captured_chunk(many):
    """A chunk of many rows over parts of the keys, captured once; each replay, with other lengths, equals the eager call."""
    n, new, cap = 2, 40, 2240
    cache = make(n, 2, 128, cap, BF16, paged=True)
    gen = torch.Generator().manual_seed(16)
    k, v = (normal(gen, n, cap, 2, 128, dtype=BF16).cuda() for _ in "kv")
    cache.append(k, v, ints([0] * n))
    q = normal(gen, n, new, 4, 128, dtype=BF16).cuda()
    lens = ints([0, 0])
    L = KV.load()
    L.owk_debug_kv8_set_many_rows(many)
    try:
        cache.attend(q, lens)  # the workspace's size
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = cache.attend(q, lens)
        for at in ([cap, 64], [0, 1280], [1920, 128], [640, cap], [64, 0]):  # whole blocks of what is held
            lens.copy_(ints(at))
            g.replay()
            torch.cuda.synchronize()
            want = cache.attend(q, lens)
            assert want.isfinite().all() and torch.equal(out, want), at
            assert all((out[b] != 0).any() == (at[b] > 0) for b in range(n)), at
    finally:
        L.owk_debug_kv8_set_many_rows(0)


@gpu
def test_other_streams_and_repeats():
    """A call on a side stream, and the same call twice: the same bits."""
    cache, model = make(4, 2, 64, 3000, F16), Model(4, 2, 64, F16)
    fill(cache, model, [2999, 1500, 64, 1])
    gen = torch.Generator().manual_seed(6)
    q = normal(gen, 4, 1, 2, 64, dtype=F16).cuda()
    lens = ints([2999, 1500, 64, 1])
    want = cache.attend(q, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q, lens)
    side.synchronize()
    assert torch.equal(got, want)
    for _ in range(3):
        assert torch.equal(cache.attend(q, lens), want)
    one = torch.cat([cache.attend(q[b:b + 1], lens[b:b + 1], seq=ints([b]), max_len=3000) for b in range(4)])
    torch.testing.assert_close(one, want, rtol=2 ** -9, atol=2 ** -9)  # another split of the keys: a step of the type or two


@gpu
@pytest.mark.parametrize("call", [
    lambda c, k, i: c.append(k, k[:, :1], i),
    lambda c, k, i: c.append(k.float(), k.float(), i),
    lambda c, k, i: c.append(k.transpose(2, 3).contiguous().transpose(2, 3), k, i),
    lambda c, k, i: c.append(k[..., :32], k[..., :32], i),
    lambda c, k, i: c.append(k, k, i.long()),
    lambda c, k, i: c.append(k, k, i.cpu()),
    lambda c, k, i: c.append(k, k, i[:1]),
    lambda c, k, i: c.append(k[0], k[0], i),
    lambda c, k, i: c.append(k, k, i, max_new=9),
    lambda c, k, i: c.append(k, k, i, off=i),
    lambda c, k, i: c.append(k[0], k[0], i, off=i, count=i),
    lambda c, k, i: c.attend(k[:, :, :1], i),
    lambda c, k, i: c.attend(k, i, out=k[:, :1]),
    lambda c, k, i: c.attend(k, i, out=k.double()),
    lambda c, k, i: c.attend(k, i, out=k[:, :1].expand_as(k)),
    lambda c, k, i: c.attend(k, i, scale=math.nan),
    lambda c, k, i: c.attend(k, i, seq=i.long()),
    lambda c, k, i: c.attend(torch.cat([k, k]), torch.cat([i, i])),
    lambda c, k, i: c.read(i.long(), 4),
    lambda c, k, i: KV.Cache(1, 1, 96, 64),
    lambda c, k, i: KV.Cache(1, 1, 64, 64, torch.float32),
    lambda c, k, i: KV.Cache.of(c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, max_blocks=9),
    lambda c, k, i: KV.Cache.of(c.k, c.v.transpose(2, 3), c.k_scale, c.v_scale, c.k_tail, c.v_tail).append(k, k, i),
])
def test_refused_calls(call):
    cache = make(2, 2, 64, 128, F16)
    k, i = torch.zeros((2, 3, 2, 64), dtype=F16, device="cuda"), ints([0, 0])
    before = cache.k_tail.clone()
    with pytest.raises(ValueError):
        call(cache, k, i)
    assert torch.equal(cache.k_tail, before)
