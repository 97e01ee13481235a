"""What the operators of voxtral_b200_serve.h refuse, and the 64-bit statement of the 4-bit format. No GPU."""
import ctypes as C
import math

import pytest
import torch

import serve_plain as plain


@pytest.fixture(scope="module")
def serve(pkg):
    import sys
    return sys.modules[pkg.__name__ + ".serve"]


def _cache(serve, seqs=2, kv_heads=2, head_dim=64, capacity=32):
    """A cache as far as the binding's checks go: its handle leads nowhere."""
    c = serve.KV4Cache.__new__(serve.KV4Cache)
    c.L, c.seqs, c.kv_heads, c.head_dim, c.capacity, c.h = serve.serve_lib(), seqs, kv_heads, head_dim, capacity, 1
    c.close = lambda: None
    return c


def _a(serve, *shape, dtype="float32", strides=None):
    return serve.DeviceArray(4096, shape, dtype, strides)


def test_open_refuses_sizes(serve):
    for args in ((1, 1, 100, 8), (1, 1, 0, 8), (1, 1, 320, 8), (0, 1, 64, 8), (1, 0, 64, 8), (1, 1, 64, 0), (70000, 1, 64, 8), (1, 1, 64, (1 << 30) + 1)):
        with pytest.raises(RuntimeError, match="has to be|have to be"):
            serve.KV4Cache(*args)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="sm_100 GPU is required"):
            serve.KV4Cache(1, 1, 64, 8)


def test_append_refuses_arrays(serve):
    c, k = _cache(serve), _a(serve, 2, 3, 2, 64)
    at = _a(serve, 2, dtype="int32")
    c.append_call(k, k, at)
    for bad in (_a(serve, 2, 3, 2, 32), _a(serve, 1, 3, 2, 64), _a(serve, 2, 3, 4, 64), _a(serve, 2, 3, 2, 64, dtype="float64"),
                _a(serve, 2, 3, 2, 64, strides=(768, 256, 128, 2)), _a(serve, 6, 2, 64)):
        with pytest.raises(ValueError):
            c.append_call(bad, bad, at)
    with pytest.raises(ValueError, match="one type"):
        c.append_call(k, _a(serve, 2, 3, 2, 64, dtype="bfloat16"), at)
    for bad in (_a(serve, 2), _a(serve, 3, dtype="int32"), _a(serve, 2, dtype="int32", strides=(2,))):
        with pytest.raises(ValueError):
            c.append_call(k, k, bad)
        with pytest.raises(ValueError):
            c.read_call(k, k, at, rows=bad)
    with pytest.raises(ValueError, match="GPU"):
        c.append_call(torch.zeros(2, 3, 2, 64), torch.zeros(2, 3, 2, 64), torch.zeros(2, dtype=torch.int32))
    c.h = None
    with pytest.raises(ValueError, match="closed"):
        c.append_call(k, k, at)


def test_attention_refuses_arrays(serve):
    c, q, at = _cache(serve), _a(serve, 2, 3, 6, 64), _a(serve, 2, dtype="int32")
    lse, mass = _a(serve, 2, 3, 6), _a(serve, 2, 2, 32)
    c.attention_call(q, q, at, lse=lse, mass_in=mass, mass_out=mass)
    for kw in ({"lse": _a(serve, 2, 6, 3)}, {"lse": lse, "mass_out": _a(serve, 2, 2, 31)}, {"mass_out": mass}, {"lse": lse, "mass_out": _a(serve, 2, 2, 32, dtype="bfloat16")},
               {"lse": lse, "mass_out": _a(serve, 2, 2, 32, strides=(128, 64, 1))}):
        with pytest.raises(ValueError):
            c.attention_call(q, q, at, **kw)
    with pytest.raises(ValueError, match="multiple"):
        c.attention_call(_a(serve, 2, 3, 3, 64), _a(serve, 2, 3, 3, 64), at)
    with pytest.raises(ValueError):
        c.attention_call(q, _a(serve, 2, 3, 6, 64, dtype="bfloat16"), at)
    with pytest.raises(ValueError):
        c.attention_call(_a(serve, 6, 6, 64), q, at)


def test_evict_refuses_arrays(serve):
    c, at, mass = _cache(serve), _a(serve, 2, dtype="int32"), _a(serve, 2, 2, 32)
    kept = _a(serve, 2, 2, 8, dtype="int32")
    c.evict_call(c, at, at, mass, mass, kept, keep=8)
    c.evict_call(c, at, at, mass, _a(serve, 2, 2, 8), kept, keep=8)
    c.evict_call(c, at, at, mass, None, kept, keep=8)
    for args in ((at, at, _a(serve, 2, 2, 31), mass, kept), (at, at, mass, _a(serve, 2, 2, 9), kept), (at, at, mass, mass, _a(serve, 2, 2, 9, dtype="int32")),
                 (at, _a(serve, 3, dtype="int32"), mass, mass, kept)):
        with pytest.raises(ValueError):
            c.evict_call(c, *args, keep=8)


def test_logprobs_refuses_arrays(pkg, serve):
    x, tok, out = _a(serve, 4, 100), _a(serve, 4, dtype="int32"), _a(serve, 4)
    pkg.token_logprobs_call(x, tok, out, out, _a(serve, 4, 5, dtype="int32"), _a(serve, 4, 5))
    for args in ((_a(serve, 400), tok, out), (_a(serve, 4, 100, dtype="int32"), tok, out), (_a(serve, 4, 100, strides=(200, 2)), tok, out), (x, _a(serve, 4), out),
                 (x, tok, _a(serve, 5)), (x, tok, out, _a(serve, 4, 1)), (x, tok, out, out, _a(serve, 4, 33, dtype="int32")), (x, tok, out, out, _a(serve, 4, 5)),
                 (x, tok, out, out, _a(serve, 4, 5, dtype="int32"), _a(serve, 4, 6)), (_a(serve, 4, 3), tok, out, out, _a(serve, 4, 5, dtype="int32"))):
        with pytest.raises(ValueError):
            pkg.token_logprobs_call(*args)


def test_c_calls_refuse_before_they_touch_a_gpu(serve):
    L = serve.serve_lib()
    err = lambda: L.vb200_serve_error().decode()  # noqa: E731
    assert L.vb200_kv4_append(None, None, None) == -1 and "no cache" in err()
    assert L.vb200_kv4_read(None, None, None) == -1
    assert L.vb200_kv4_attention(None, None, None) == -1
    assert L.vb200_kv4_evict(None, None, None, None) == -1
    assert L.vb200_kv4_status(None) == -1 and L.vb200_kv4_bytes(None) == 0
    L.vb200_kv4_close(None)
    assert L.vb200_token_logprobs(None, None) == -1
    good = dict(logits=4096, type=0, rows=2, vocab=10, row_stride=10, tokens=4096, logprobs=4096, entropy=None, top=0, top_ids=None, top_logprobs=None)
    for change, word in (({"type": 3}, "fp32"), ({"logits": 4098}, "aligned"), ({"logits": 4097, "type": 1}, "aligned"), ({"rows": -1}, "rows"), ({"vocab": 0}, "vocab"),
                         ({"top": 33}, "top"), ({"top": 11}, "top"), ({"top": -1}, "top"), ({"tokens": None}, "tokens"), ({"logits": None}, "no logits")):
        a = serve._LogprobsArgs(**dict(good, **change))
        assert L.vb200_token_logprobs(C.byref(a), None) == -1 and word in err(), (change, err())
    assert L.vb200_token_logprobs(C.byref(serve._LogprobsArgs(**dict(good, rows=0))), None) == 0


def test_statement_of_the_format():
    x = torch.zeros(2, 64)
    x[0, :8] = torch.tensor([0.25, 0.26, 0.75, 1.25, 2.5, 3.5, 5.0, 7.9])
    x[0, 40] = math.inf
    x[1, 33] = 2.0 ** -140
    y = plain.rounded(x)
    assert y[0, :8].tolist() == [0.0, 0.5, 1.0, 1.0, 2.0, 4.0, 4.0, 6.0]
    assert torch.isnan(y[0, 32:]).all() and (y[0, 8:32] == 0).all() and (y[1] == 0).all()
    z = torch.randn(100, 96)
    r = plain.rounded(z).unflatten(-1, (-1, 32))
    most = z.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    # half a step of the coarsest level, or what lies beyond 6
    assert ((r - z.double().unflatten(-1, (-1, 32))).abs() <= most / 4 + 1e-12).all()
    assert torch.equal(plain.rounded(r.flatten(-2)), r.flatten(-2))


def test_statement_of_attention_and_eviction():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=g) for s in ((3, 4, 32), (2, 7, 32), (2, 7, 32)))
    out, lse, mass = plain.attention(q, k, v, 7, 3, 0.2)
    for i in range(3):
        for u in range(4):
            s = torch.softmax((k[u // 2, :5 + i] @ q[i, u] * 0.2).double(), 0)
            assert torch.allclose(out[i, u], s @ v[u // 2, :5 + i].double(), atol=1e-6)
    assert torch.allclose(mass.sum(1), torch.full((2,), 6.0, dtype=torch.float64))
    out, lse, _ = plain.attention(q, k, v, 2, 3, 0.2)                 # the first row sees nothing
    assert (out[0] == 0).all() and torch.isinf(lse[0]).all() and torch.isfinite(lse[1:]).all()
    assert plain.kept(torch.tensor([1.0, 5.0, 5.0, 2.0, 5.0, 0.0]), 6, 3, 1, 0) == [1, 2, 5]
    assert plain.kept(torch.tensor([math.nan, 1.0, math.nan, 0.0]), 4, 2, 0, 0) == [1, 3]
