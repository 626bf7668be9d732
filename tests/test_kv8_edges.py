"""The 8-bit key/value cache at the edges of its types and tables: what a row sees of blocks of very different size, of
hidden blocks, of values that are not finite, in both forms of attention (16-row and 128-row tiles). Oracle and bounds are
test_kv8.py's."""
import contextlib
import math
import threading

import pytest
import torch

import owk_kv8 as KV
from test_kv8 import BF16, BLOCK, F16, Model, Raw, _batch, _desc, _params, attend, check_attend, fill, ints, make, normal

gpu = pytest.mark.gpu
FORMS = [32, 1 << 30]  # rows of a head above which tiles of 128 rows are taken


@contextlib.contextmanager
def form(cache, rows):
    L = KV.load()
    cache._ws.clear()
    L.owk_debug_kv8_set_many_rows(rows)
    try:
        yield
    finally:
        L.owk_debug_kv8_set_many_rows(0)
        cache._ws.clear()


def one_head(dtype, k, v, paged=False):
    """A cache and model of one sequence that hold k, v [tokens, heads, dim] (given in 64 bits, rounded to dtype)."""
    n, h, d = k.shape
    cache, model = make(1, h, d, n, dtype, paged=paged), Model(1, h, d, dtype)
    k, v = k.to(dtype), v.to(dtype)
    cache.append(k[None].cuda(), v[None].cuda(), ints([0]))
    model.append(0, 0, k, v)
    return cache, model


def spread(gen, *shape):
    """Magnitudes in [1, 2), signs at random, in 64 bits."""
    x = torch.rand(shape, generator=gen, dtype=torch.float64)
    return (1 + x) * (2.0 * (torch.rand(shape, generator=gen) < 0.5) - 1)


# ---------------------------------------------------------------------------------------------------
# hidden blocks
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("rows", FORMS)
@pytest.mark.parametrize("dim,dtype", [(64, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("causal", [False, True])
def test_nothing_is_seen_of_a_hidden_block(dim, dtype, rows, causal):
    """Whatever the pool's blocks hold, a table entry out of the pool adds nothing: the same bits."""
    n, new, h = 3 * BLOCK + 7, 40, 2
    gen = torch.Generator().manual_seed(31)
    table = torch.tensor([[3, 1, 2, 4]], dtype=torch.int32, device="cuda")  # block 0 of the pool is no sequence's
    cache, model = KV.Cache(1, h, dim, 256, dtype, "cuda", n_blocks=6, table=table), Model(1, h, dim, dtype)
    k, v = (normal(gen, n, h, dim, dtype=dtype) for _ in "kv")
    if dtype == BF16:
        v = (v.double() * 2.0 ** -60).to(dtype)
    cache.append(k[None].cuda(), v[None].cuda(), ints([0]))
    model.append(0, 0, k, v)
    table[0, 1] = -1
    q = normal(gen, 1, new, h, dim, dtype=dtype).cuda()
    at = n - new if causal else n
    cache.k[0], cache.v[0] = 77, -33
    outs = []
    with form(cache, rows):
        for scale in (0.0, 1.0, 2.0 ** 100, math.inf, math.nan):
            cache.k_scale[0], cache.v_scale[0] = scale, scale
            outs.append(cache.attend(q, ints([at]), causal=causal, out=torch.zeros_like(q, dtype=torch.float32)))
    for x in outs[1:]:
        assert torch.equal(x, outs[0])
    keep = torch.cat([torch.arange(0, 64), torch.arange(128, n)])
    kk, vv = model.held(0, "k")[keep], model.held(0, "v")[keep]
    seen = [int((keep <= at + i).sum()) if causal else keep.numel() for i in range(new)]
    want, bound = attend(q[0].cpu(), kk, vv, dim ** -0.5, seen, torch.float32)
    # (the bound's blocks of 64 start at other tokens than the cache's, with at most twice the spread of probabilities)
    assert ((outs[0][0].cpu().double() - want).abs() <= 2 * bound).all()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_values_near_the_end_of_f32(dim):
    """Tiles of 128 rows over whole blocks: the sum of a row's weighted values passes the range of f32, the output does not."""
    gen = torch.Generator().manual_seed(54)
    n, new = 256, 40
    v, k = spread(gen, n, 1, dim).abs() * 2.0 ** 125, 0.1 * spread(gen, n, 1, dim)
    cache, model = one_head(BF16, k, v)
    q = spread(gen, 1, new, 1, dim).to(BF16)
    want, bound = attend(q[0], model.held(0, "k"), model.held(0, "v"), dim ** -0.5, [n] * new, torch.float32)
    with form(cache, 32):
        got = cache.attend(q.cuda(), ints([n]), out=torch.empty((1, new, 1, dim), device="cuda"))
    assert ((got[0].cpu().double() - want).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("n", [64, 50])
def test_equal_values(dim, dtype, n):
    """Weights are divided by their own sum as they were rounded: tokens of equal values give that value to f32's last bits, over
    a block of codes and over a tail, however few of them a row sees."""
    gen = torch.Generator().manual_seed(55)
    k = 0.5 * spread(gen, n, 2, dim)
    v = torch.full((n, 2, dim), 0.75, dtype=torch.float64)
    cache, model = one_head(dtype, k, v)
    check_attend(cache, model, [0], [n], 1, True, scale=0.1, out_type=torch.float32)
    check_attend(cache, model, [n - 12], [12], 2, True, scale=0.1, out_type=torch.float32)


# ---------------------------------------------------------------------------------------------------
# tails
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("before", [0, 64])
def test_later_tokens_of_the_tail(dim, before):
    """Causal rows over a bf16 tail: the size of later tokens' keys and values is nothing to a row."""
    gen = torch.Generator().manual_seed(43)
    new = 40
    n = before + new
    v, k = spread(gen, n, 1, dim), 0.3 * spread(gen, n, 1, dim)
    v[before + 20:] *= 2.0 ** 40
    k[before + 30:] *= 2.0 ** 60
    cache, model = one_head(BF16, k, v)
    check_attend(cache, model, [before], [new], 1, True, scale=1.0, out_type=torch.float32)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_one_large_key_of_the_tail(dim):
    """A key of the tail that no row attends to, far larger than the others."""
    gen = torch.Generator().manual_seed(44)
    n, new = 50, 40
    v, k = spread(gen, n, 1, dim), 0.3 * spread(gen, n, 1, dim)
    k[5, :, 0] = -2.0 ** 23  # (the bound stays finite)
    v[5] = 2.0 ** 40
    cache, model = one_head(BF16, k, v)
    q = 0.3 * torch.randn((new, 1, dim), generator=gen)
    q[:, :, 0] = 1.0
    check_attend(cache, model, [n], [new], 1, False, rows=[q.to(BF16)], scale=1.0, out_type=torch.float32)


# ---------------------------------------------------------------------------------------------------
# queries that are not finite
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("rows", FORMS)
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("n", [0, 20, 64, 100])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(dim, dtype, rows, n, bad):
    """A row with such a query is NaN if it sees anything, and no other row is."""
    gen = torch.Generator().manual_seed(46)
    new = 40
    k, v = spread(gen, max(n, 1), 1, dim), spread(gen, max(n, 1), 1, dim)
    k[..., 3] = k[..., 3].abs()  # all scores of one sign
    cache, _ = one_head(dtype, k, v)
    q = normal(gen, 1, new, 1, dim, dtype=dtype).cuda()
    for q_rows, count in ((q, new), (q[:, :3].contiguous(), 3)):
        with form(cache, rows):
            clean = cache.attend(q_rows, ints([n]))
            x = q_rows.clone()
            x[0, 1, 0, 3] = bad
            got = cache.attend(x, ints([n]))
        others = [i for i in range(count) if i != 1]
        assert clean.isfinite().all() and got[0, others].isfinite().all()
        assert got[0, 1].isnan().all() if n else not got[0, 1].any()


# ---------------------------------------------------------------------------------------------------
# queries
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power,scale", [(-120, 0.125), (-110, 0.125), (110, 0.125), (126, 4.0), (126, -4.0)])
@pytest.mark.parametrize("n", [64, 100, 150])
def test_queries_of_any_size(dim, power, scale, n):
    """Tiny queries of large keys and large queries of tiny keys: the same scores."""
    gen = torch.Generator().manual_seed(45)
    new = 40
    k, v = 0.5 * spread(gen, n, 1, dim) * 2.0 ** -min(power, 118), spread(gen, n, 1, dim)
    cache, model = one_head(BF16, k, v)
    q = 0.5 * spread(gen, new, 1, dim) * 2.0 ** power
    check_attend(cache, model, [n], [new], 1, False, rows=[q.to(BF16)], scale=scale, out_type=torch.float32)
    check_attend(cache, model, [n], [2], 1, False, rows=[q[:2].to(BF16)], scale=scale, out_type=torch.float32)


# ---------------------------------------------------------------------------------------------------
# blocks of very different size
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,ratio", [(F16, 20), (F16, 24), (F16, 26), (F16, 28), (BF16, 30), (BF16, 45), (BF16, 60)])
@pytest.mark.parametrize("order", ["small first", "large first", "in turn"])
def test_large_values_of_small_weight(dim, dtype, ratio, order):
    """A block whose values are 2^ratio larger and whose weights as much smaller adds as much as the others."""
    gen = torch.Generator().manual_seed(ratio)
    sizes = {"small first": [0, 1], "large first": [1, 0], "in turn": [0, 1, 0, 0, 1]}[order]
    n, new = 64 * len(sizes) + 3, 40
    big = torch.tensor(sizes + [0]).repeat_interleave(64)[:n, None, None]
    v = spread(gen, n, 1, dim) * torch.where(big > 0, 2.0 ** (ratio // 2), 2.0 ** (ratio // 2 - ratio))
    k = 0.2 * spread(gen, n, 1, dim)
    k[:, :, 0] = torch.where(big[..., 0] > 0, -(ratio + 0.3) * math.log(2), 0.0)  # with q[0] = 1 and scale 1: the score's level
    cache, model = one_head(dtype, k, v)
    q = 0.3 * torch.randn((new, 1, dim), generator=gen)
    q[:, :, 0] = 1.0
    q[1::4, :, 0] = 1.25  # rows that see less and more of them
    q[2::4, :, 0] = 0.75
    check_attend(cache, model, [n], [new], 1, False, rows=[q.to(dtype)], scale=1.0, out_type=torch.float32)
    check_attend(cache, model, [n - new], [new], 1, True, rows=[q.to(dtype)], scale=1.0, out_type=torch.float32)
    check_attend(cache, model, [n], [2], 1, False, rows=[q[:2].to(dtype)], scale=1.0, out_type=torch.float32)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_values_of_zero_under_a_large_weight(dim):
    """One block takes nearly all of the weight and has values of zero: the rest is what the output is made of."""
    gen = torch.Generator().manual_seed(41)
    n, new = 4 * 64, 48
    v, k = spread(gen, n, 1, dim), 0.2 * spread(gen, n, 1, dim)
    k[:64, :, 0] = 24.0
    v[:64] = 0.0
    cache, model = one_head(BF16, k, v)
    q = 0.3 * torch.randn((new, 1, dim), generator=gen)
    q[:, :, 0] = 1.0
    check_attend(cache, model, [n], [new], 1, False, rows=[q.to(BF16)], scale=1.0, out_type=torch.float32)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("low,high", [(-40, 40), (-70, 80), (-100, 110)])
def test_a_block_of_other_rows(dim, low, high):
    """Causal rows of one tile: the size of a block that some of them see is nothing to those before it."""
    gen = torch.Generator().manual_seed(42)
    n, at = 3 * 64, 40
    v, k = spread(gen, n, 1, dim), 0.3 * spread(gen, n, 1, dim)
    v[:64] *= 2.0 ** low
    v[64:128] *= 2.0 ** high
    cache, model = one_head(BF16, k, v)
    check_attend(cache, model, [at], [n - at], 1, True, scale=1.0, out_type=torch.float32)

@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("rows", FORMS)
def test_rows_do_not_depend_on_each_other(dim, dtype, rows):
    """A row's bits are the same whatever the rows beside it are."""
    gen = torch.Generator().manual_seed(53)
    n, new = 300, 40
    v, k = spread(gen, n, 1, dim), 0.5 * spread(gen, n, 1, dim)
    v *= 2.0 ** torch.randint(-12, 12, (6, 1, 1), generator=gen).repeat_interleave(64, 0)[:n]
    cache, _ = one_head(dtype, k, v)
    q = 0.5 * spread(gen, 1, new, 1, dim)
    with form(cache, rows):
        want = cache.attend(q.to(dtype).cuda(), ints([n]), scale=1.0)
        for other in (0.0, 12.0, math.nan):
            x = q.clone()
            x[:, ::3] *= other
            got = cache.attend(x.to(dtype).cuda(), ints([n]), scale=1.0)
            for i in (1, 2):
                assert torch.equal(got[:, i::3], want[:, i::3]), (other, i)


# ---------------------------------------------------------------------------------------------------
# keys and values that are not finite
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_complete_block_that_is_not_finite(dim, dtype, which, bad):
    """It is NaN to the rows that see any of it: not to causal rows before it, nor to another head or sequence."""
    lens = [230, 230]
    cache, model = make(2, 2, dim, 320, dtype, paged=True), Model(2, 2, dim, dtype)
    gen = torch.Generator().manual_seed(47)
    for s, n in enumerate(lens):
        k, v = (normal(gen, n, 2, dim, dtype=dtype) for _ in "kv")
        if s == 0:
            (k if which == "k" else v)[100, 1, 7] = bad
        cache.append(k[None].cuda(), v[None].cuda(), ints([0]), seq=ints([s]))
        model.append(s, 0, k, v)
    check_attend(cache, model, lens, [40, 40], 1, False)
    check_attend(cache, model, lens, [2, 2], 2, False)
    check_attend(cache, model, [20, 20], [210, 210], 1, True)  # rows before it, in it and behind it
    for at in (62, 63, 64, 127, 128):
        check_attend(cache, model, [at, at], [lens[0] - at] * 2, 1, True, max_len=256)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("new", [1, 40])
def test_parts_that_are_not_finite(dim, dtype, which, new):
    """One part of a long sequence's keys is NaN: the join keeps it."""
    lens = [6000, 6000]
    cache, model = make(2, 1, dim, 6016, dtype, paged=True), Model(2, 1, dim, dtype)
    gen = torch.Generator().manual_seed(48)
    for s, n in enumerate(lens):
        k, v = (normal(gen, n, 1, dim, dtype=dtype) for _ in "kv")
        if s == 0:
            (k if which == "k" else v)[4321, 0, 7] = math.nan
        cache.append(k[None].cuda(), v[None].cuda(), ints([0]), seq=ints([s]))
        model.append(s, 0, k, v)
    check_attend(cache, model, lens, [new, new], 1, False)


@gpu
@pytest.mark.parametrize("rows", FORMS)
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("before", [0, 64])
def test_a_tail_token_that_is_not_finite(dim, dtype, rows, which, before):
    """Only later causal rows see it, in its own head and sequence."""
    new, odd = 50, before + 30
    lens = [before, before]
    cache, model = make(2, 2, dim, 128, dtype), Model(2, 2, dim, dtype)
    fill(cache, model, [before + new] * 2)
    gen = torch.Generator().manual_seed(49)
    q = normal(gen, 2, new, 2, dim, dtype=dtype).cuda()
    with form(cache, rows):
        clean = cache.attend(q, ints(lens), causal=True)
        if which == "k":
            cache.k_tail[1, 0, odd % BLOCK, 5] = math.nan
        else:
            cache.v_tail[1, 0, 5, odd % BLOCK] = math.inf
        got = cache.attend(q, ints(lens), causal=True)
    sees = [lens[1] + i >= odd for i in range(new)]
    assert clean.isfinite().all()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :, 1], clean[1, :, 1])
    for i in range(new):
        if not sees[i]:
            assert torch.equal(got[1, i, 0], clean[1, i, 0]), i
        else:
            assert not got[1, i, 0, 5].isfinite(), i
            assert which == "v" or got[1, i, 0].isnan().all(), i


# ---------------------------------------------------------------------------------------------------
# the 128-row form in the calls that the 16-row one is tested in
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("rows", FORMS)
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_many_rows_over_the_queries(dim, dtype, rows):
    """Outputs where the queries are, in one part and in several that are joined."""
    for lens, cap in (([190, 65], 200), ([5000, 3100], 5056)):
        cache, model = make(2, 2, dim, cap, dtype), Model(2, 2, dim, dtype)
        fill(cache, model, lens)
        gen = torch.Generator().manual_seed(50)
        q = normal(gen, 2, 70, 4, dim, dtype=dtype).cuda()
        with form(cache, rows):
            want = cache.attend(q, ints(lens))
            assert want.isfinite().all()
            assert torch.equal(cache.attend(q, ints(lens), out=q), want)


@gpu
@pytest.mark.parametrize("rows", FORMS)
def test_many_rows_of_hidden_pages_and_bad_sequences(rows):
    cache, model = make(3, 2, 64, 256, F16, paged=True), Model(3, 2, 64, F16)
    lens, new = [200, 140, 70], 40
    fill(cache, model, lens)
    good = cache.table.clone()
    gen = torch.Generator().manual_seed(51)
    q = normal(gen, 3, new, 2, 64, dtype=F16)
    for bad in (-1, 10 ** 9, cache.k.shape[0]):
        cache.table.copy_(good)
        cache.table[0, 1] = bad
        with form(cache, rows):
            out = cache.attend(q.cuda(), ints(lens), seq=ints([0, 7, 2])).cpu().double()
        keep = torch.cat([torch.arange(0, 64), torch.arange(128, 200)])
        want, bound = attend(q[0], model.held(0, "k")[keep], model.held(0, "v")[keep], 0.125, [keep.numel()] * new, F16)
        # (the bound's blocks of 64 start at other tokens than the cache's, with at most twice the spread of probabilities)
        assert ((out[0] - want).abs() <= 2 * bound).all()
        assert not out[1].any()
        want, bound = attend(q[2], model.held(2, "k"), model.held(2, "v"), 0.125, [70] * new, F16)
        assert ((out[2] - want).abs() <= bound).all()
    cache.table[0] = -1  # nothing is held but the tail
    with form(cache, rows):
        out = cache.attend(q.cuda(), ints(lens)).cpu().double()
    want, bound = attend(q[0], model.held(0, "k")[192:], model.held(0, "v")[192:], 0.125, [8] * new, F16)
    assert ((out[0] - want).abs() <= bound).all()


# ---------------------------------------------------------------------------------------------------
# the binding
# ---------------------------------------------------------------------------------------------------
@gpu
def test_tensors_of_a_cache_are_fixed():
    """A cache's tensors change in place alone: another one under the same name would not be read."""
    cache, model = make(2, 2, 64, 200, F16, paged=True), Model(2, 2, 64, F16)
    fill(cache, model, [190, 65])
    for name in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "table"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, getattr(cache, name).clone())
    with pytest.raises(AttributeError):
        cache.n_heads = 1
    cache.table.copy_(cache.table.flip(0))
    k, _ = cache.read(ints([128, 64]), 64, seq=ints([1, 0]))
    for s in range(2):
        assert torch.equal(k[s].cpu(), model.held(s, "k")[:64].float().half()), s


# ---------------------------------------------------------------------------------------------------
# arguments out of range
# ---------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("call", [
    lambda c, k, i: c.attend(k, i, max_len=1 << 31),
    lambda c, k, i: c.attend(k, i, max_len=-(1 << 40)),
    lambda c, k, i: c.attend(k, i, scale=1e60),
    lambda c, k, i: c.attend(k[0], i[:1], off=i, max_new=1 << 40),
    lambda c, k, i: c.append(k[0], k[0], i[:1], off=i, max_new=1 << 31),
    lambda c, k, i: c.append(k, k, i, max_new=-(1 << 33)),
    lambda c, k, i: c.read(i, -1),
    lambda c, k, i: c.read(i, (1 << 32) + 1),
])
def test_arguments_out_of_range(call):
    cache = make(2, 2, 64, 128, F16)
    k, i = torch.zeros((2, 3, 2, 64), dtype=F16, device="cuda"), ints([0, 0])
    with pytest.raises(ValueError):
        call(cache, k, i)


def test_the_switch_of_the_form_is_a_threads_own():
    """owk_debug_kv8_set_many_rows on one thread changes no other thread's calls."""
    L = Raw()
    d, b, p = _desc(n_seqs=1, n_heads=1, n_blocks=4096, max_blocks=4096), _batch(n=1, max_new=40), _params(n_q_heads=1)
    sizes = []

    def other():
        sizes.append(L.owk_kv8_attend_workspace(d, b, p))

    want = [L.owk_kv8_attend_workspace(d, b, p)]
    try:
        for rows in (32, 1 << 30):
            KV.load().owk_debug_kv8_set_many_rows(rows)
            want.append(L.owk_kv8_attend_workspace(d, b, p))
            t = threading.Thread(target=other)
            t.start()
            t.join()
    finally:
        KV.load().owk_debug_kv8_set_many_rows(0)
    assert want[1] != want[2]  # the switch does something here
    assert sizes == [want[0]] * 2
