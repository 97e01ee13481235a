"""Binding of the operators for servers of language models (include/voxtral_b200_serve.h): a key/value cache in 4
bits, attention over it, eviction from it, log probabilities of tokens. All of them work on device memory.

    cache = KV4Cache(seqs=8, kv_heads=8, head_dim=128, capacity=32768)
    cache.append(k, v, lengths)                        # lengths [seqs]: the tokens in the cache, the new ones counted
    cache.attention(q, out, lengths, lse=lse, mass_in=mass, mass_out=mass)
    cache.evict(cache, lengths, lengths, mass, mass, kept, keep=8192, recent=1024, first=4)
    token_logprobs(logits, tokens, logprobs, entropy, top_ids, top_logprobs)

Arrays are torch CUDA tensors, or anything else with data_ptr(), shape, stride() and dtype as they have them (DeviceArray makes one of a
pointer). They are not copied, cast or made contiguous: what a call cannot take it refuses with ValueError. Calls are
queued on `stream` (a cudaStream_t as a number; 0: the default stream), not on torch's current stream unless that is what is given,
and return at once; the arrays have to live until the work is done.

Every method has a `..._call` form, which checks its arguments once and returns a Call: call(stream) queues the same work again,
as a loop over tokens does.
"""
import ctypes as C
import math

from .lm import lm_lib

TYPES = {"float32": 0, "bfloat16": 1, "float16": 2}


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("type", C.c_int), ("seq", C.c_longlong), ("row", C.c_longlong), ("head", C.c_longlong)]


class _AppendArgs(C.Structure):
    _fields_ = [("lengths", C.c_void_p), ("rows", C.c_void_p), ("max_rows", C.c_int), ("k", _Rows), ("v", _Rows)]


class _AttentionArgs(C.Structure):
    _fields_ = [("lengths", C.c_void_p), ("rows", C.c_void_p), ("max_rows", C.c_int), ("heads", C.c_int), ("scale", C.c_float), ("q", _Rows), ("out", _Rows),
                ("lse", C.c_void_p), ("mass_in", C.c_void_p), ("mass_out", C.c_void_p)]


class _EvictArgs(C.Structure):
    _fields_ = [("lengths", C.c_void_p), ("new_lengths", C.c_void_p), ("mass", C.c_void_p), ("new_mass", C.c_void_p), ("new_mass_ld", C.c_longlong),
                ("kept", C.c_void_p), ("keep", C.c_int), ("recent", C.c_int), ("first", C.c_int)]


class _LogprobsArgs(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("type", C.c_int), ("rows", C.c_int), ("vocab", C.c_int), ("row_stride", C.c_longlong), ("tokens", C.c_void_p),
                ("logprobs", C.c_void_p), ("entropy", C.c_void_p), ("top", C.c_int), ("top_ids", C.c_void_p), ("top_logprobs", C.c_void_p)]


_libs = {}


def serve_lib(path=None):
    """The shared library with these entry points (the language models' one)."""
    L = lm_lib(path)
    if id(L) not in _libs:
        for name, res, args in (
                ("vb200_serve_error", C.c_char_p, []),
                ("vb200_kv4_open", C.c_void_p, [C.c_int] * 4),
                ("vb200_kv4_close", None, [C.c_void_p]),
                ("vb200_kv4_bytes", C.c_size_t, [C.c_void_p]),
                ("vb200_kv4_status", C.c_int, [C.c_void_p]),
                ("vb200_kv4_append", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p]),
                ("vb200_kv4_read", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p]),
                ("vb200_kv4_attention", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p]),
                ("vb200_kv4_evict", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
                ("vb200_token_logprobs", C.c_int, [C.c_void_p, C.c_void_p])):
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _libs[id(L)] = L
    return L


class DeviceArray:
    """Device memory of somebody else's as an array: pointer, shape, type ("float32", "bfloat16", "float16", "int32"), strides in
    elements (dense where they are not given)."""

    def __init__(self, pointer, shape, dtype="float32", strides=None, device=None):
        self._pointer, self.shape, self.dtype, self.device = int(pointer), tuple(shape), dtype, device
        if strides is None:
            strides, n = [], 1
            for s in reversed(self.shape):
                strides.insert(0, n)
                n *= s
        self._strides = tuple(strides)

    def data_ptr(self):
        return self._pointer

    def stride(self):
        return self._strides


def _dtype(a):
    return str(a.dtype).split(".")[-1]


def _place(a):
    """The number of the GPU that an array says it lies on, None if it says nothing."""
    d = getattr(a, "device", None)
    if d is None:
        return None
    if getattr(d, "type", None) != "cuda":
        raise ValueError("arrays have to lie on a GPU")
    return d.index


def _dense(a, name, shape, dtype):
    if a is None:
        return None
    if tuple(a.shape) != tuple(shape) or _dtype(a) != dtype:
        raise ValueError(f"{name} has to be {dtype} of shape {tuple(shape)}: got {_dtype(a)} of shape {tuple(a.shape)}")
    n = 1
    for size, stride in zip(reversed(tuple(a.shape)), reversed(tuple(a.stride()))):
        if size > 1 and stride != n and 0 not in shape:
            raise ValueError(f"{name} has to be dense")
        n *= size
    return a.data_ptr()


def _rows(a, name, seqs, rows, heads, head_dim):
    """[seqs, rows, heads, head_dim] with values of a head side by side."""
    if tuple(a.shape) != (seqs, rows, heads, head_dim):
        raise ValueError(f"{name} has to be of shape {(seqs, rows, heads, head_dim)}: got {tuple(a.shape)}")
    if _dtype(a) not in TYPES:
        raise ValueError(f"{name} has to be float32, bfloat16 or float16: got {_dtype(a)}")
    s = a.stride()
    if s[3] != 1:
        raise ValueError(f"the values of a head of {name} have to lie side by side")
    return _Rows(a.data_ptr(), TYPES[_dtype(a)], s[0], s[1], s[2])


class Call:
    """A checked call: call(stream) queues it. It keeps the arrays that it is about."""
    __slots__ = ("_fn", "_caches", "_args", "_lib", "_keep")

    def __init__(self, L, fn, caches, args, keep):
        self._lib, self._fn, self._caches, self._args, self._keep = L, fn, caches, C.byref(args), (args, keep)

    def __call__(self, stream=0):
        handles = [c.h for c in self._caches]
        if None in handles:
            raise ValueError("the cache is closed")
        if self._fn(*handles, self._args, stream) != 0:
            raise RuntimeError(self._lib.vb200_serve_error().decode())


class KV4Cache:
    """Keys and values of `seqs` sequences of up to `capacity` tokens, in 4 bits, on the current GPU. Calls on one cache are made one after
    another: on one stream, or on streams that events put in order."""

    def __init__(self, seqs, kv_heads, head_dim, capacity, lib_path=None):
        self.L = serve_lib(lib_path)
        self.seqs, self.kv_heads, self.head_dim, self.capacity = seqs, kv_heads, head_dim, capacity
        self.h = None
        self.h = self.L.vb200_kv4_open(seqs, kv_heads, head_dim, capacity)
        if not self.h:
            raise RuntimeError(self.L.vb200_serve_error().decode())

    def bytes(self):
        return self.L.vb200_kv4_bytes(self.h)

    def check(self):
        """Waits for the device; raises where a bounded wait inside a kernel has run out since the last check."""
        s = self.L.vb200_kv4_status(self.h)
        if s:
            raise RuntimeError(f"a bounded wait ran out on the device (status {s})" if s > 0 else self.L.vb200_serve_error().decode())

    def _open(self):
        if not self.h:
            raise ValueError("the cache is closed")

    def _spans(self, lengths, rows, arrays):
        places = {_place(a) for a in arrays if a is not None} - {None}
        if len(places) > 1:
            raise ValueError("the arrays lie on different GPUs")
        return _dense(lengths, "lengths", (self.seqs,), "int32"), _dense(rows, "rows", (self.seqs,), "int32")

    def _move(self, fn, k, v, lengths, rows):
        self._open()
        if _dtype(k) != _dtype(v):
            raise ValueError("k and v have to be of one type")
        ln, rw = self._spans(lengths, rows, (k, v, lengths, rows))
        n = k.shape[1] if len(k.shape) == 4 else 0
        shape = (self.seqs, n, self.kv_heads, self.head_dim)
        a = _AppendArgs(ln, rw, n, _rows(k, "k", *shape), _rows(v, "v", *shape))
        return Call(self.L, fn, (self,), a, (k, v, lengths, rows))

    def append_call(self, k, v, lengths, rows=None):
        return self._move(self.L.vb200_kv4_append, k, v, lengths, rows)

    def append(self, k, v, lengths, rows=None, stream=0):
        """k, v [seqs, max_rows, kv_heads, head_dim] into the cache, as its last tokens. rows [seqs]: how many of them are real."""
        self.append_call(k, v, lengths, rows)(stream)

    def read_call(self, k, v, lengths, rows=None):
        return self._move(self.L.vb200_kv4_read, k, v, lengths, rows)

    def read(self, k, v, lengths, rows=None, stream=0):
        """The last tokens of the cache, as the values that it holds, out into k, v."""
        self.read_call(k, v, lengths, rows)(stream)

    def attention_call(self, q, out, lengths, scale=None, rows=None, lse=None, mass_in=None, mass_out=None):
        self._open()
        if len(q.shape) != 4:
            raise ValueError("q has to be [seqs, rows, heads, head_dim]")
        n, heads = q.shape[1], q.shape[2]
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"q has {heads} heads: not a multiple of the cache's {self.kv_heads}")
        if _dtype(q) != _dtype(out):
            raise ValueError("q and out have to be of one type")
        ln, rw = self._spans(lengths, rows, (q, out, lengths, rows, lse, mass_in, mass_out))
        shape, mass = (self.seqs, n, heads, self.head_dim), (self.seqs, self.kv_heads, self.capacity)
        if mass_out is not None and lse is None:
            raise ValueError("mass_out needs lse")
        a = _AttentionArgs(ln, rw, n, heads, 1.0 / math.sqrt(self.head_dim) if scale is None else scale, _rows(q, "q", *shape), _rows(out, "out", *shape),
                           _dense(lse, "lse", shape[:3], "float32"), _dense(mass_in, "mass_in", mass, "float32"), _dense(mass_out, "mass_out", mass, "float32"))
        return Call(self.L, self.L.vb200_kv4_attention, (self,), a, (q, out, lengths, rows, lse, mass_in, mass_out))

    def attention(self, q, out, lengths, scale=None, rows=None, lse=None, mass_in=None, mass_out=None, stream=0):
        """Causal attention of q [seqs, rows, heads, head_dim], the queries of the last tokens, into out. scale: 1 / sqrt(head_dim) where
        it is not given; lse [seqs, rows, heads]; mass_in, mass_out [seqs, kv_heads, capacity]."""
        self.attention_call(q, out, lengths, scale, rows, lse, mass_in, mass_out)(stream)

    def evict_call(self, into, lengths, new_lengths, mass, new_mass, kept, keep, recent=0, first=0):
        self._open()
        into._open()
        self._spans(lengths, None, (lengths, new_lengths, mass, new_mass, kept))
        ln, nl = _dense(lengths, "lengths", (self.seqs,), "int32"), _dense(new_lengths, "new_lengths", (self.seqs,), "int32")
        ld = keep
        if new_mass is not None and new_mass.shape[-1] in (self.capacity, into.capacity):
            ld = max(keep, new_mass.shape[-1])
        a = _EvictArgs(ln, nl, _dense(mass, "mass", (self.seqs, self.kv_heads, self.capacity), "float32"),
                       _dense(new_mass, "new_mass", (self.seqs, self.kv_heads, ld), "float32"), ld,
                       _dense(kept, "kept", (self.seqs, self.kv_heads, keep), "int32"), keep, recent, first)
        return Call(self.L, self.L.vb200_kv4_evict, (self, into), a, (lengths, new_lengths, mass, new_mass, kept))

    def evict(self, into, lengths, new_lengths, mass, new_mass, kept, keep, recent=0, first=0, stream=0):
        """Sequences of more than `keep` tokens are cut to that many, by mass; what stays goes into the first slots of `into` (a
        cache like this one, or this one). new_lengths, new_mass ([.., keep], or [.., the capacity of either cache], or None) and kept [seqs,
        kv_heads, keep] are results."""
        self.evict_call(into, lengths, new_lengths, mass, new_mass, kept, keep, recent, first)(stream)

    def close(self):
        if self.h:
            self.L.vb200_kv4_close(self.h)
            self.h = None

    def __del__(self):
        if getattr(self, "h", None):
            self.close()


def token_logprobs_call(logits, tokens, logprobs, entropy=None, top_ids=None, top_logprobs=None, lib_path=None):
    L = serve_lib(lib_path)
    if len(logits.shape) != 2 or _dtype(logits) not in TYPES:
        raise ValueError("logits have to be [rows, vocab] of float32, bfloat16 or float16")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride()[1] != 1:
        raise ValueError("the logits of a row have to lie side by side")
    arrays = (logits, tokens, logprobs, entropy, top_ids, top_logprobs)
    if len({_place(a) for a in arrays if a is not None} - {None}) > 1:
        raise ValueError("the arrays lie on different GPUs")
    tops = [a for a in (top_ids, top_logprobs) if a is not None]
    top = tops[0].shape[1] if tops and len(tops[0].shape) == 2 else 0
    if tops and not 1 <= top <= min(32, vocab):
        raise ValueError("top_ids and top_logprobs have to be [rows, 1 .. 32], at most vocab")
    a = _LogprobsArgs(logits.data_ptr(), TYPES[_dtype(logits)], rows, vocab, logits.stride()[0], _dense(tokens, "tokens", (rows,), "int32"),
                      _dense(logprobs, "logprobs", (rows,), "float32"), _dense(entropy, "entropy", (rows,), "float32"), top,
                      _dense(top_ids, "top_ids", (rows, top), "int32"), _dense(top_logprobs, "top_logprobs", (rows, top), "float32"))
    return Call(L, L.vb200_token_logprobs, (), a, arrays)


def token_logprobs(logits, tokens, logprobs, entropy=None, top_ids=None, top_logprobs=None, stream=0, lib_path=None):
    """Out of logits [rows, vocab]: the log probability of tokens[r] (int32), the entropy, the most probable tokens ([rows, 1 .. 32]), each
    where there is an array for it. A token outside the vocabulary has NaN."""
    token_logprobs_call(logits, tokens, logprobs, entropy, top_ids, top_logprobs, lib_path)(stream)
