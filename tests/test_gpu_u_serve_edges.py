"""The operators for servers of language models (include/voxtral_b200_serve.h) where they could go wrong: rows that differ within a warp, values far apart,
weights far below the largest, sizes around the borders between kernels' schemes. Against the same in 64 bits."""
import math

import pytest
import torch

import serve_plain as plain
from test_gpu_t_serve import TYPES, _fill, _gen, _held, _ints, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,n,rows,heads,kv_heads", [("f32", 7001, 100, 160, 160), ("bf16", 7001, 100, 160, 160), ("f16", 2050, 3, 12, 2)])
def test_rows_of_a_warp_whose_scores_rise_differently(pkg, dtype, n, rows, heads, kv_heads):
    """Halfway the scores rise by 0, 5 or 80 binary orders, the next row's by another number: rows that are taken together change their
    references at different times, and sums are put aside between."""
    g, t, d, half = _gen(73), TYPES[dtype], 32, n // 2
    k, v = torch.zeros(1, n, kv_heads, d, device="cuda", dtype=t), _randn(g, 1, n, kv_heads, d, dtype=t).abs()
    k[:, half:, :, 0] = 4.0
    cache, at = _fill(pkg, k, v, n, [n])
    q = torch.zeros(1, rows, heads, d, device="cuda", dtype=t)
    for i in range(rows):
        for u in range(heads // kv_heads):
            q[0, i, u::heads // kv_heads, 0] = (0.0, 5.0, 80.0)[(i + u) % 3] * math.log(2.0) / 4.0
    out, lse = torch.full_like(q, 3.0), torch.full((1, rows, heads), 4.0, device="cuda")
    cache.attention(q, out, at, scale=1.0, lse=lse)
    cache.check()
    vv = _held(v, None)[0].repeat_interleave(heads // kv_heads, 0)       # [heads, n, d]
    early, late = vv[:, :half].sum(1)[None], vv[:, half:].cumsum(1)[:, -rows:].transpose(0, 1)
    rise = q[0, :, :, 0].double() * 4.0                                  # natural
    w = torch.exp(-rise)
    count = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] + (n - rows - half + 1)
    z = half * w + count
    want = (early * w[..., None] + late) / z[..., None]
    # as for rows that rise alike: a score's roundings, twice in a weight, exponentials and terms, sums a unit for each 16 tokens and term, FP16's
    # smallest step for every early token, the result's own rounding
    score = rise * (2.0 ** -22 + 10 * 2.0 ** -23)
    limit = want * (2 * score[..., None] + 2.0 ** -19 + (n / 8 + 16) * 2.0 ** -23 + (2.0 ** -11 if dtype == "bf16" else 0.0) + torch.finfo(t).eps / 2)
    limit = limit + early * 2.0 ** -32 / count[..., None]
    assert ((out[0].double() - want).abs() <= limit).all()
    total = torch.log(z) + rise
    assert ((lse[0].double() - total).abs() <= score + 2.0 ** -18 + total.abs() * 2.0 ** -23).all()


def test_host_memory_is_refused_wherever_it_is_given(pkg):
    """Every pointer of every call in turn: from C nothing else stands between it and the kernels."""
    import ctypes as C
    import sys
    serve = sys.modules[pkg.__name__ + ".serve"]
    L = serve.serve_lib()
    host = torch.zeros(1 << 16)
    p, h = (lambda t: t.data_ptr()), host.data_ptr()
    cache = pkg.KV4Cache(2, 2, 64, 32)
    k, q, at = torch.zeros(2, 3, 2, 64, device="cuda"), torch.zeros(2, 3, 4, 64, device="cuda"), _ints(3, 3)
    out, lse, mass = torch.zeros_like(q), torch.zeros(2, 3, 4, device="cuda"), torch.zeros(2, 2, 32, device="cuda")
    kept, x = torch.zeros(2, 2, 8, dtype=torch.int32, device="cuda"), torch.zeros(2, 100, device="cuda")
    rows = lambda data, heads: serve._Rows(data, 0, 3 * heads * 64, heads * 64, 64)  # noqa: E731
    move = dict(lengths=p(at), rows=p(at), max_rows=3, k=rows(p(k), 2), v=rows(p(k), 2))
    att = dict(lengths=p(at), rows=p(at), max_rows=3, heads=4, scale=1.0, q=rows(p(q), 4), out=rows(p(out), 4), lse=p(lse), mass_in=p(mass), mass_out=p(mass))
    ev = dict(lengths=p(at), new_lengths=p(at), mass=p(mass), new_mass=p(mass), new_mass_ld=32, kept=p(kept), keep=8, recent=2, first=1)
    lp = dict(logits=p(x), type=0, rows=2, vocab=100, row_stride=100, tokens=p(at), logprobs=p(lse), entropy=p(lse), top=1, top_ids=p(kept), top_logprobs=p(lse))
    new = torch.zeros_like(mass)
    calls = [(fn, (cache.h,), serve._AppendArgs, move, {"lengths": h, "rows": h, "k": rows(h, 2), "v": rows(h, 2)}) for fn in (L.vb200_kv4_append, L.vb200_kv4_read)]
    calls += [(L.vb200_kv4_attention, (cache.h,), serve._AttentionArgs, att, {"lengths": h, "rows": h, "q": rows(h, 4), "out": rows(h, 4), "lse": h, "mass_in": h, "mass_out": h}),
              (L.vb200_kv4_evict, (cache.h, cache.h), serve._EvictArgs, dict(ev, new_mass=p(new)), {"lengths": h, "new_lengths": h, "mass": h, "new_mass": h, "kept": h}),
              (L.vb200_token_logprobs, (), serve._LogprobsArgs, lp, {"logits": h, "tokens": h, "logprobs": h, "entropy": h, "top_ids": h, "top_logprobs": h})]
    for fn, handles, args, good, bad in calls:
        for name, value in bad.items():
            assert fn(*handles, C.byref(args(**dict(good, **{name: value}))), None) == -1, (fn, name)
            assert "not lie" in L.vb200_serve_error().decode() and name in L.vb200_serve_error().decode()
        assert fn(*handles, C.byref(args(**good)), None) == 0, L.vb200_serve_error()
    # host memory that the device reaches is no fault: lengths may be there
    pinned = torch.full((2,), 3, dtype=torch.int32).pin_memory()
    assert L.vb200_kv4_append(cache.h, C.byref(serve._AppendArgs(**dict(move, lengths=pinned.data_ptr()))), None) == 0
    torch.cuda.synchronize()
    cache.check()
