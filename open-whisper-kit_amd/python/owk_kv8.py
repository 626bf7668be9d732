"""Binding of include/owk_kv8.h: keys and values held in 8 bits, on torch tensors of one GPU.

    cache = Cache(n_seqs=4, n_heads=8, head_dim=64, max_tokens=4096, device="cuda")
    cache.append(k, v, lens)                    # k, v: [4, n, 8, 64], their tokens go behind lens[b]
    out = cache.attend(q, lens, causal=True)    # q: [4, n, 8 * group, 64] -> the same shape
    lens += n

Tensors of entries are padded, [entry, row, head, head_dim] with `count` rows each (None: all), or joined,
[row, head, head_dim] with entry b's rows at off[b] .. off[b + 1] - 1; the innermost dimension is contiguous.
Index tensors (lens, seq, off, count, first) are int32 on the cache's device and are read there: nothing
here waits for the GPU, and every call can be captured into a graph. Calls go to the current stream of
the cache's device. One layer of a model is one Cache; layers share lens. Bad arguments raise ValueError.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch  # before the library: both use one HIP runtime

import owk

BLOCK = 64
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class CacheDesc(C.Structure):
    _fields_ = [("device", C.c_int), ("dtype", C.c_int), ("head_dim", C.c_int), ("n_heads", C.c_int), ("n_seqs", C.c_int),
                ("n_blocks", C.c_int), ("max_blocks", C.c_int), ("k", C.c_void_p), ("v", C.c_void_p),
                ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("k_tail", C.c_void_p), ("v_tail", C.c_void_p),
                ("table", C.c_void_p)]


class Batch(C.Structure):
    _fields_ = [("n", C.c_int), ("max_new", C.c_int), ("rows", C.c_int64), ("lens", C.c_void_p), ("seq", C.c_void_p),
                ("off", C.c_void_p), ("count", C.c_void_p)]


class Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("entry", C.c_int64), ("row", C.c_int64), ("head", C.c_int64)]


class AttendParams(C.Structure):
    _fields_ = [("n_q_heads", C.c_int), ("causal", C.c_int), ("out_type", C.c_int), ("max_len", C.c_int), ("scale", C.c_float)]


# the same three structures as bytes: packing is several times quicker than filling a ctypes.Structure, and a call of one
# token is as long on the host as on the GPU
_BATCH, _ROWS, _PARAMS = struct.Struct("iiqPPPP").pack, struct.Struct("Pqqq").pack, struct.Struct("iiiif").pack

_lib = None


def load():
    global _lib
    if _lib is None:
        L = owk.load()
        vp = C.c_void_p
        L.owk_kv8_append.argtypes = [vp, vp, vp, vp, vp]
        L.owk_kv8_attend.argtypes = [vp, vp, vp, vp, vp, vp, C.c_size_t, vp]
        L.owk_kv8_attend_workspace.argtypes = [vp, vp, vp]
        L.owk_kv8_attend_workspace.restype = C.c_size_t
        L.owk_kv8_read.argtypes = [vp, C.c_int, C.c_int, vp, vp, vp, vp, vp, vp]
        L.owk_kv8_error.restype = C.c_char_p
        _lib = L
    return _lib


def _check(rc):
    if rc:
        msg = load().owk_kv8_error().decode("utf-8", "replace")
        raise ValueError(msg) if rc == -1 else RuntimeError(msg)


class Cache:
    """The cache of one layer: `n_seqs` sequences of up to `max_tokens` tokens (rounded up to whole blocks). With
    `table` (int32 [n_seqs, blocks], kept, read at every call) sequences take their blocks from a pool of `n_blocks`. Contents of
    the tensors may be changed in place; the tensors themselves are the cache's for good."""

    def __init__(self, n_seqs, n_heads, head_dim, max_tokens, dtype=torch.float16, device="cuda", n_blocks=None, table=None):
        blocks = table.shape[1] if table is not None else -(-int(max_tokens) // BLOCK)
        pool = n_blocks if n_blocks is not None else n_seqs * blocks

        def new(shape, t):
            return torch.zeros(shape, dtype=t, device=device)

        self._bind(new((pool, n_heads, BLOCK, head_dim), torch.int8), new((pool, n_heads, head_dim, BLOCK), torch.int8),
                   new((pool, n_heads), torch.float32), new((pool, n_heads), torch.float32),
                   new((n_seqs, n_heads, BLOCK, head_dim), dtype), new((n_seqs, n_heads, head_dim, BLOCK), dtype), table, blocks)

    @classmethod
    def of(cls, k, v, k_scale, v_scale, k_tail, v_tail, table=None, max_blocks=None):
        """A cache over tensors that the caller made, in the layouts of owk_kv8.h. Without a table the pool is cut into
        equal runs of `max_blocks` blocks (None: as many as fit)."""
        self = cls.__new__(cls)
        blocks = table.shape[1] if table is not None else max_blocks or k.shape[0] // max(1, k_tail.shape[0])
        self._bind(k, v, k_scale, v_scale, k_tail, v_tail, table, blocks)
        return self

    def _bind(self, k, v, k_scale, v_scale, k_tail, v_tail, table, blocks):
        pool, heads, _, dim = k.shape
        seqs, dtype, dev = k_tail.shape[0], k_tail.dtype, k.device
        want = ((k, torch.int8, (pool, heads, BLOCK, dim)), (v, torch.int8, (pool, heads, dim, BLOCK)),
                (k_scale, torch.float32, (pool, heads)), (v_scale, torch.float32, (pool, heads)),
                (k_tail, dtype, (seqs, heads, BLOCK, dim)), (v_tail, dtype, (seqs, heads, dim, BLOCK)))
        for x, t, shape in want + (((table, torch.int32, (seqs, blocks)),) if table is not None else ()):
            if x.dtype != t or tuple(x.shape) != shape or x.device != dev or not x.is_contiguous():
                raise ValueError(f"a cache tensor is {x.dtype} {tuple(x.shape)} on {x.device}, wanted contiguous {t} {shape} on {dev}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a cache of {dtype}: float16 or bfloat16 are supported")
        if dim not in (64, 128):
            raise ValueError(f"head_dim {dim}: 64 or 128 are supported")
        if dev.type != "cuda":
            raise ValueError(f"the cache is on {dev}: a GPU is needed")
        if table is None and not 0 < seqs * blocks <= pool:
            raise ValueError(f"{seqs} sequences of {blocks} blocks do not fit a pool of {pool}")
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail, self.table = (
            k, v, k_scale, v_scale, k_tail, v_tail, table)
        self.device, self.dtype, self.n_heads, self.head_dim = dev, dtype, heads, dim
        self.n_seqs, self.max_tokens = seqs, blocks * BLOCK
        self.desc = CacheDesc(dev.index, _TYPES[dtype], dim, heads, seqs, pool, blocks, k.data_ptr(), v.data_ptr(),
                              k_scale.data_ptr(), v_scale.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr(),
                              table.data_ptr() if table is not None else None)
        self._at = C.addressof(self.desc)
        self._dev = dev.index
        self._L = load()
        self._ws = {}

    def __setattr__(self, name, value):
        # calls use the addresses that the cache was made of: another tensor would be ignored, and the old one's memory be
        # given away under them
        if name in self.__dict__:
            raise AttributeError(f"{name} of a cache is fixed: copy into it, or make another with Cache.of")
        object.__setattr__(self, name, value)

    def _index(self, name, x, n):
        if x is None:
            return 0
        if x.dtype is not torch.int32 or x.get_device() != self._dev or x.shape != (n,) or not x.is_contiguous():
            raise ValueError(f"{name} is {x.dtype} {tuple(x.shape)} on {x.device}, wanted contiguous int32 ({n},) on {self.device}")
        return x.data_ptr()

    def _batch(self, shape, lens, seq, off, count, max_new):
        n = lens.shape[0] if lens.dim() else 0
        if seq is None and n > self.n_seqs:
            raise ValueError(f"{n} entries, and the cache has {self.n_seqs} sequences")
        rows = 0
        if off is None:
            if len(shape) != 4 or shape[0] != n:
                raise ValueError(f"a padded tensor of {n} entries is [{n}, rows, heads, {self.head_dim}], got {tuple(shape)}")
            if max_new is None:
                max_new = shape[1]
            elif max_new > shape[1]:
                raise ValueError(f"max_new {max_new} passes the tensor's {shape[1]} rows")
        else:
            if len(shape) != 3 or count is not None:
                raise ValueError(f"joined tensors are [rows, heads, {self.head_dim}] without count, got {tuple(shape)}")
            rows = shape[0]
            if max_new is None:
                max_new = rows
        at = (self._index("lens", lens, n), self._index("seq", seq, n), self._index("off", off, n + 1), self._index("count", count, n))
        try:
            return _BATCH(n, max_new, rows, *at), n, max_new
        except struct.error:
            raise ValueError(f"max_new {max_new} is out of range") from None

    def _rows(self, name, x, shape, heads, dtype):
        s = x.stride()
        if x.dtype is not dtype or x.get_device() != self._dev or shape[-1] != self.head_dim or shape[-2] != heads:
            raise ValueError(f"{name} is {x.dtype} {tuple(shape)} on {x.device}, wanted {dtype} [.., {heads}, {self.head_dim}] "
                             f"on {self.device}")
        if s[-1] != 1:
            raise ValueError(f"the innermost dimension of {name} is not contiguous")
        return _ROWS(x.data_ptr(), s[0] if len(s) == 4 else 0, s[-3], s[-2])

    def _stream(self):
        return torch._C._cuda_getCurrentRawStream(self._dev)

    def append(self, k, v, lens, seq=None, off=None, count=None, max_new=None):
        """Store the entries' tokens behind the lens[b] that their sequences hold (or from an earlier multiple of 64 on)."""
        shape = k.shape
        b, _, _ = self._batch(shape, lens, seq, off, count, max_new)
        if shape != v.shape:
            raise ValueError(f"k is {tuple(shape)} and v is {tuple(v.shape)}")
        kr, vr = self._rows("k", k, shape, self.n_heads, self.dtype), self._rows("v", v, shape, self.n_heads, self.dtype)
        if k.numel():
            _check(self._L.owk_kv8_append(self._at, b, kr, vr, self._stream()))

    def attend(self, q, lens, seq=None, off=None, count=None, max_new=None, max_len=0, scale=None, causal=False, out=None):
        """softmax(scale * q . k) . v over what the sequences hold: tokens [0, lens[b]), or with causal, for row i,
        [0, lens[b] + i] (its own tokens appended before). scale None: 1 / sqrt(head_dim). `max_len`: no sequence holds
        more (a hint for splitting the work). `out`: a tensor like q (q itself, too), or float32; rows that are no entry's stay as they are
        (undefined in a new tensor). Weights and some queries have fewer bits than 32, also into float32: owk_kv8.h says how many. No
        gradients."""
        shape = q.shape
        b, n, max_new = self._batch(shape, lens, seq, off, count, max_new)
        heads = shape[-2]
        if heads < 1 or heads % self.n_heads:
            raise ValueError(f"{heads} query heads are no multiple of {self.n_heads} key/value heads")
        qr = self._rows("q", q, shape, heads, self.dtype)
        if out is None:
            out = torch.empty_like(q)
            if 0 in out.stride():
                out = torch.empty(shape, dtype=q.dtype, device=q.device)
        elif out.shape != shape:
            raise ValueError(f"out is {tuple(out.shape)} and q is {tuple(shape)}")
        elif any(i > 1 and t == 0 for i, t in zip(shape, out.stride())):
            raise ValueError("rows of out lie on each other")
        of = out.dtype
        orow = self._rows("out", out, shape, heads, of if of is torch.float32 else self.dtype)
        try:
            p = _PARAMS(heads, 1 if causal else 0, _TYPES[of], max_len, self.head_dim ** -0.5 if scale is None else scale)
        except (struct.error, OverflowError):
            raise ValueError(f"max_len {max_len} or scale {scale} is out of range") from None
        if q.numel():
            need = self._ws.get((n, max_new, heads, max_len))
            if need is None:  # a function of these sizes alone
                if len(self._ws) >= 1024:
                    self._ws.clear()
                need = self._ws[(n, max_new, heads, max_len)] = self._L.owk_kv8_attend_workspace(self._at, b, p)
            ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            _check(self._L.owk_kv8_attend(self._at, b, p, qr, orow, ws.data_ptr() if need else None, need, self._stream()))
        return out

    def read(self, lens, max_tokens, seq=None, first=None):
        """Tokens first[b] (None: 0) .. + max_tokens of sequences that hold lens[b]: (k, v), each [entry, token, head,
        head_dim] in the cache's 16-bit type, zeros from lens[b] on."""
        n = lens.shape[0] if lens.dim() else 0
        if seq is None and n > self.n_seqs:
            raise ValueError(f"{n} entries, and the cache has {self.n_seqs} sequences")
        if not 0 <= max_tokens < 1 << 31:
            raise ValueError(f"max_tokens {max_tokens} is out of range")
        h, d = self.n_heads, self.head_dim
        kv = self.k_tail.new_empty((2, n, max_tokens, h, d))
        k, v = kv.unbind(0)
        i = self._index("lens", lens, n), self._index("seq", seq, n), self._index("first", first, n)
        if kv.numel():
            at, one = kv.data_ptr(), max_tokens * h * d
            _check(self._L.owk_kv8_read(self._at, n, max_tokens, *i, _ROWS(at, one, h * d, d),
                                        _ROWS(at + 2 * n * one, one, h * d, d), self._stream()))
        return k, v
