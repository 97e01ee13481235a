"""The operators for servers of language models (include/voxtral_b200_serve.h) where they could go wrong: rows that differ within a warp, values far apart,
weights far below the largest, sizes around the borders between kernels' schemes. Against the same in 64 bits."""
import math

import pytest
import torch

import serve_plain as plain
from test_gpu_t_serve import TYPES, _check_logprobs, _fill, _gen, _held, _ints, _randn

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


def _check_by_component(out, lse, q, k, v, rows, scale, dtype, mass=None, before=None):
    """Against 64 bits, every result within its own roundings: those of sum p |v| and of sum |q k|, whatever the largest |v| and |k| of the
    cache are. One sequence; k, v [H, n, D] as they are held."""
    n, heads, h, d = k.shape[1], q.shape[2], k.shape[0], k.shape[-1]
    g = heads // h
    sees = torch.arange(n, device="cuda")[None] < torch.arange(n - rows + 1, n + 1, device="cuda")[:, None]
    want_mass = torch.zeros(h, n, dtype=torch.float64, device="cuda")
    mass_limit = torch.zeros_like(want_mass)
    for u in range(heads):
        kk, vv, qq = k[u // g].double(), v[u // g].double(), q[0, :rows, u].double()
        s = torch.where(sees, qq @ kk.T * scale, -math.inf)
        total = torch.logsumexp(s, 1, keepdim=True)
        p = torch.exp(s - total)
        want = p @ vv
        sums = torch.where(sees, qq.abs() @ kk.abs().T * abs(scale), 0.0)
        # as attention_bounds derives them, of the weights that count: those of a row by their own sums of magnitudes
        score = sums * ((2 * d // 32 + 4) * 2.0 ** -23 + 2.0 ** -22 + 4 * 2.0 ** -24 + 2.0 ** -21)
        of_sum = (p * score).sum(1, keepdim=True)
        weight = p * (score + of_sum + 2.0 ** -19 + (2.0 ** -11 if dtype == torch.bfloat16 else 0.0) + (n / 8 + 16) * 2.0 ** -23)
        limit = weight @ vv.abs() + want.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
        err = (out[0, :rows, u].double() - want).abs()
        assert (err <= limit).all(), (u, float((err / limit).max()))
        assert ((lse[0, :rows, u, None].double() - total).abs() <= of_sum + 2.0 ** -18 + total.abs() * 2.0 ** -23).all()
        want_mass[u // g] += p.sum(0)
        mass_limit[u // g] += (p * (score + of_sum + 2.0 ** -18)).sum(0)
    if mass is not None:
        assert ((mass[0, :, :n].double() - want_mass).abs() <= mass_limit + 2.0 ** -24 * (want_mass + before[0, :, :n])).all()


# rows, heads, KV heads, head_dim, tokens, capacity: a few rows; many, as a unit alone, in parts and in a last round of parts
FAR = [(1, 4, 1, 64, 400, 400), (5, 2, 1, 128, 300, 300), (3, 4, 2, 96, 200, 200), (80, 2, 1, 64, 200, 200000), (70, 4, 2, 128, 5000, 120000), (90, 2, 2, 96, 9000, 120000),
       (65, 150, 150, 32, 2100, 2100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads,kv_heads,dim,n,capacity", FAR)
def test_large_values_of_tokens_that_weigh_little(pkg, rows, heads, kv_heads, dim, n, capacity, dtype):
    """Every eighth token's values are 2^40 times the others' (2^14 in fp16, which has no more) and its weight 2^-45 (2^-19)."""
    g, t = _gen(79), TYPES[dtype]
    far = 14 if dtype == "f16" else 40
    k, v = torch.zeros(1, n, kv_heads, dim, device="cuda"), _randn(g, 1, n, kv_heads, dim)
    k[:, ::8, :, 0] = -4.0
    k[:, ::8, :, 1] = 0.5
    v = v / 64.0 if dtype == "f16" else v
    v[:, ::8] = (v[:, ::8] * 2.0 ** far).clamp(-60000.0, 60000.0) if dtype == "f16" else v[:, ::8] * 2.0 ** far
    k, v = k.to(t), v.to(t)
    cache, at = _fill(pkg, k, v, capacity, [n])
    q = (_randn(g, 1, rows, heads, dim) * 0.1).to(t)
    q[..., 0] = (far + 5) * math.log(2.0) / 4.0
    out, lse = torch.full_like(q, 3.0), torch.full((1, rows, heads), 4.0, device="cuda")
    cache.attention(q, out, at, scale=1.0, lse=lse)
    cache.check()
    _check_by_component(out, lse, q, _held(k, None)[0], _held(v, None)[0], rows, 1.0, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("big", [20, 50, 100, 120])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,n,capacity", FAR)
def test_large_values_that_a_row_does_not_see(pkg, rows, heads, kv_heads, dim, n, capacity, big, dtype):
    """The portion's tokens have values 2^big times the cache's, each four times the one before: rows that see none of a token's have nothing of it."""
    g, t = _gen(83), TYPES[dtype]
    k, v = _randn(g, 1, n, kv_heads, dim), _randn(g, 1, n, kv_heads, dim)
    for i in range(min(rows - 1, 3)):
        v[:, n - 1 - i] *= 2.0 ** (big - 2 * i)
    k, v = k.to(t), v.to(t)
    cache, at = _fill(pkg, k, v, capacity, [n])
    q = _randn(g, 1, rows, heads, dim, dtype=t)
    out, lse = torch.full_like(q, 3.0), torch.full((1, rows, heads), 4.0, device="cuda")
    cache.attention(q, out, at, lse=lse)
    cache.check()
    _check_by_component(out, lse, q, _held(k, None)[0], _held(v, None)[0], rows, dim ** -0.5, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,n,capacity", [x for x in FAR if x[3] >= 64])
def test_keys_of_very_different_magnitude(pkg, rows, heads, kv_heads, dim, n, capacity, dtype):
    """Every seventh token's keys are 2^45 in dims that the queries leave out and the last one's 2^100, so that scores are as the others' keys
    make them. With masses, into what was there."""
    g, t = _gen(97), TYPES[dtype]
    k, v, q = _randn(g, 1, n, kv_heads, dim), _randn(g, 1, n, kv_heads, dim), _randn(g, 1, rows, heads, dim)
    k[:, ::7, :, 32:] *= 2.0 ** 45
    k[:, n - 1, :, 32:] *= 2.0 ** 55
    q[..., 32:] = 0.0
    k, v, q = k.to(t), v.to(t), q.to(t)
    cache, at = _fill(pkg, k, v, capacity, [n])
    out, lse = torch.full_like(q, 3.0), torch.full((1, rows, heads), 4.0, device="cuda")
    mass = torch.rand(1, kv_heads, capacity, generator=g, device="cuda")
    before = mass.clone()
    cache.attention(q, out, at, lse=lse, mass_in=mass, mass_out=mass)
    cache.check()
    assert torch.equal(mass[..., n:], before[..., n:])
    before[..., n - rows:] = 0.0
    _check_by_component(out, lse, q, _held(k, None)[0], _held(v, None)[0], rows, dim ** -0.5, t, mass.double() - before.double(), before)


def test_blocks_of_zeros(pkg):
    """Blocks of zeros beside others, and nothing but zeros: no scale of theirs stands in anything's way."""
    g = _gen(89)
    for rows in (1, 3):
        n, h, heads, d = 300, 2, 4, 128
        k, v = _randn(g, 1, n, h, d), _randn(g, 1, n, h, d)
        k[:, ::3, :, :32], v[:, ::5, :, 64:], v[:, 7::11] = 0.0, 0.0, -0.0
        v[:, :, 1, 32:64] = 0.0
        cache, at = _fill(pkg, k, v, n, [n])
        gk, gv = torch.empty_like(k), torch.empty_like(v)
        cache.read(gk, gv, at)
        assert torch.equal(gk.double(), plain.rounded(k)) and torch.equal(gv.double(), plain.rounded(v))
        q = _randn(g, 1, rows, heads, d)
        out, lse = torch.full_like(q, 3.0), torch.empty(1, rows, heads, device="cuda")
        cache.attention(q, out, at, lse=lse)
        _check_by_component(out, lse, q, _held(k, None)[0], _held(v, None)[0], rows, d ** -0.5, torch.float32)
        assert (out[0, :, 2:, 32:64] == 0).all()


@pytest.mark.parametrize("dtype,small", [("f32", 8), ("f32", 20), ("f32", 90), ("bf16", 8), ("bf16", 40), ("f16", 8)])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,n,capacity", FAR)
def test_small_queries(pkg, rows, heads, kv_heads, dim, n, capacity, dtype, small):
    """Queries of 2^-small, of a model that normalises them or far smaller: weights come out nearly even, in tiles that end inside a sequence too."""
    g, t = _gen(103), TYPES[dtype]
    k, v, q = _randn(g, 1, n, kv_heads, dim, dtype=t), _randn(g, 1, n, kv_heads, dim, dtype=t), (_randn(g, 1, rows, heads, dim) * 2.0 ** -small).to(t)
    cache, at = _fill(pkg, k, v, capacity, [n])
    for scale in (dim ** -0.5, 2.0 ** -60):
        out, lse = torch.full_like(q, 3.0), torch.full((1, rows, heads), 4.0, device="cuda")
        mass = torch.zeros(1, kv_heads, capacity, device="cuda")
        cache.attention(q, out, at, scale=scale, lse=lse, mass_out=mass)
        cache.check()
        _check_by_component(out, lse, q, _held(k, None)[0], _held(v, None)[0], rows, scale, t, mass, torch.zeros_like(mass))


@pytest.mark.parametrize("rows,heads,kv_heads,dim,n,capacity,large", [
    (3, 4, 2, 96, 200, 200, 95), (3, 4, 2, 96, 200, 200, -80), (80, 2, 1, 64, 200, 200000, 115), (80, 2, 1, 64, 200, 200000, -80), (70, 4, 2, 128, 5000, 120000, 115)])
def test_masses_of_large_keys_and_small_queries(pkg, rows, heads, kv_heads, dim, n, capacity, large):
    """Keys of 2^large, queries of 2^-large: scores are ordinary numbers, and so are all of their parts where factors meet first."""
    g = _gen(101)
    k, v, q = _randn(g, 1, n, kv_heads, dim) * 2.0 ** large, _randn(g, 1, n, kv_heads, dim), _randn(g, 1, rows, heads, dim) * 2.0 ** -large
    cache, at = _fill(pkg, k, v, capacity, [n])
    out, lse = torch.full_like(q, 3.0), torch.full((1, rows, heads), 4.0, device="cuda")
    mass = torch.zeros(1, kv_heads, capacity, device="cuda")
    cache.attention(q, out, at, lse=lse, mass_out=mass)
    cache.check()
    _check_by_component(out, lse, q, _held(k, None)[0], _held(v, None)[0], rows, dim ** -0.5, torch.float32, mass, torch.zeros_like(mass))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads", [(1, 300), (100, 160)])
def test_weights_far_below_the_largest(pkg, rows, heads, dtype):
    """Eight tokens at the front and 65528 that are 20 below them: together they count, each of them 2^-29. More heads than CTAs that run at
    once: a warp or two goes through a whole sequence."""
    t, n, d, tops = TYPES[dtype], 65536, 32, 8
    k, v = torch.zeros(1, n, 1, d, device="cuda", dtype=t), torch.ones(1, n, 1, d, device="cuda", dtype=t)
    k[:, 0:32 * tops:32, :, 0], v[:, 0:32 * tops:32] = 4.0, 0.0
    cache, at = _fill(pkg, k.expand(1, n, heads, d), v.expand(1, n, heads, d), n, [n])
    q = torch.zeros(1, rows, heads, d, device="cuda", dtype=t)
    q[..., 0] = 5.0
    out, lse = torch.full_like(q, 3.0), torch.empty(1, rows, heads, device="cuda")
    cache.attention(q, out, at, scale=1.0, lse=lse)
    cache.check()
    count = torch.arange(n - rows + 1, n + 1, device="cuda", dtype=torch.float64)[:, None, None] - tops
    low = math.exp(-20.0)
    want = (count * low / (tops + count * low)).expand(rows, heads, d)
    # a weight: half of FP16's smallest step, 2^-25 of 2^13 (the reference, which the first tokens are), of 2^11 where rows are many and references
    # trail by 2^4 below FP16's 2^15; a score's roundings (20 times 10 of 2^-24)
    # twice, an exponential and terms; sums: a unit for each 16 tokens and term; the result's own rounding
    relative = 2 * 20 * 10 * 2.0 ** -24 + 2.0 ** -19 + (n / 8 + 16) * 2.0 ** -23 + (2.0 ** -11 if dtype == "bf16" else 0.0)
    limit = count * (2.0 ** -38 if rows == 1 else 2.0 ** -36) / tops + want * (relative + torch.finfo(t).eps / 2) + (2.0 ** -25 if dtype == "f16" else 0.0)      # fp16: its smallest step
    err = (out[0].double() - want).abs()
    assert (err <= limit).all(), float((err / limit).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [777, 20011, 131072])
def test_entropy_of_logits_further_apart_than_the_largest_number(pkg, vocab, dtype):
    """A mask's lowest value beside logits of 1e38, in every place of a row: finite numbers, so finite entropies."""
    t = TYPES[dtype]
    x = torch.full((4, vocab), torch.finfo(t).min, device="cuda", dtype=t)
    x[0, 5] = 1e38
    x[1, vocab - 3] = 1e38
    x[2, vocab // 2:] = 1e38
    x[3, ::2] = 1e38
    ent, lp = torch.full((4,), 5.0, device="cuda"), torch.full((4,), 5.0, device="cuda")
    tokens = _ints(5, vocab - 3, vocab - 1, 0)
    pkg.token_logprobs(x, tokens, lp, ent)
    many = torch.tensor([1.0, 1.0, vocab - vocab // 2, (vocab + 1) // 2], dtype=torch.float64, device="cuda").log()
    assert torch.allclose(ent.double(), many, rtol=0.0, atol=1e-4) and torch.allclose(lp.double(), -many, rtol=0.0, atol=1e-4)


@pytest.mark.parametrize("vocab,base", [(20000, -200.0), (9001, -math.inf), (131072, -60.0)])
def test_logprobs_of_peaked_rows(pkg, vocab, base):
    """The maximum far into a row, up to 30 above the largest before it, which the same thread has read: log probabilities near 0 to fp32's own
    step, never above 0, entropies never below."""
    rows = 600
    d = torch.linspace(0.01, 30.0, rows, device="cuda")
    x = torch.full((rows, vocab), base, device="cuda")
    x[:, 0], x[:, 8192] = 0.0, d
    lp, ent, top = (torch.full(s, 5.0, device="cuda") for s in ((rows,), (rows,), (rows, 1)))
    pkg.token_logprobs(x, torch.full((rows,), 8192, dtype=torch.int32, device="cuda"), lp, ent, None, top)
    # the sum is 1 + e, e below 1: exponentials (2^-21, and 2^-23 of their argument) count with e, the sum and its logarithm with half a step each
    rest = torch.exp(-d.double()) + (vocab - 2) * torch.exp(base - d.double())
    limit = 2.0 ** -23 + rest * (2.0 ** -21 + d.double() * 2.0 ** -23)
    want = -torch.log1p(rest)
    assert ((lp.double() - want).abs() <= limit).all(), float(((lp.double() - want).abs() / limit).max())
    assert torch.equal(top[:, 0], lp) and (lp <= 0).all() and (ent >= 0).all()
    p = torch.exp(-d.double()) / (1 + rest)
    low = 0.0 if base == -math.inf else (vocab - 2) * torch.exp(base - d.double()) / (1 + rest) * (d.double() - base)
    want_ent = -want + p * d.double() + low
    assert ((ent.double() - want_ent).abs() <= limit + (p * d.double() + low) * (2.0 ** -20 + d.double() * 2.0 ** -22)).all()


@pytest.mark.parametrize("capacity", [60, 300])
def test_eviction_into_a_cache_of_another_size_and_on(pkg, capacity):
    """Masses go along into the layout of the other cache, whose attention adds to them."""
    g = _gen(107)
    s, h, heads, d, cap, keep = 2, 2, 8, 64, 200, 50
    lengths = [200, 45]
    k, v, mass = _randn(g, s, cap, h, d), _randn(g, s, cap, h, d), torch.rand(s, h, cap, generator=g, device="cuda")
    cache, at = _fill(pkg, k, v, cap, lengths)
    into, new = pkg.KV4Cache(s, h, d, capacity), torch.empty_like(at)
    new_mass, kept = torch.full((s, h, capacity), -1.0, device="cuda"), torch.empty(s, h, keep, dtype=torch.int32, device="cuda")
    cache.evict(into, at, new, mass, new_mass, kept, keep=keep, recent=10, first=2)
    assert new.tolist() == [50, 45]
    q, nk, nv = _randn(g, s, 1, heads, d), _randn(g, s, 1, h, d), _randn(g, s, 1, h, d)
    new += 1
    into.append(nk, nv, new)
    out, lse, after = torch.empty_like(q), torch.empty(s, 1, heads, device="cuda"), new_mass.clone()
    into.attention(q, out, new, lse=lse, mass_in=after, mass_out=after)
    into.check()
    for i in range(s):
        n = int(new[i])
        which = [plain.kept(mass[i, j], lengths[i], keep, 10, 2) for j in range(h)]
        hk, hv = (torch.stack([torch.cat((plain.rounded(x)[i, which[j], j], plain.rounded(y)[i, :, j])) for j in range(h)]) for x, y in ((k, nk), (v, nv)))
        was = torch.stack([torch.cat((mass[i, j, which[j]], torch.zeros(1, device="cuda"))) for j in range(h)])
        want, want_lse, want_mass = plain.attention(q[i], hk, hv, n, 1, d ** -0.5, was)
        score, result = plain.attention_bounds(q[i], hk, hv, d ** -0.5, torch.float32)
        assert ((out[i].double() - want).abs() <= result + 2.0 ** -24 * want.abs()).all()
        assert ((after[i, :, :n].double() - want_mass).abs() <= want_mass * (2 * score + 2.0 ** -20)).all()
        assert (after[i, :, n:] == -1.0).all()


def test_status_is_said_once(pkg):
    """A code where a wait that ran out leaves it (written there by another call; no wait is made to run out): check raises, then the cache goes on."""
    import ctypes as C
    cache = pkg.KV4Cache(1, 1, 64, 70)
    # the handle: planes, five sizes, workspace pointers, of which the status is the fifth; the base of it all behind two sizes
    planes, status = C.c_void_p.from_address(cache.h).value, C.c_void_p.from_address(cache.h + 56 + 32).value
    assert planes < status < planes + cache.bytes() and status % 4 == 0
    x = torch.zeros(1, 100, device="cuda")
    x[0, 61] = 1.0
    pkg.token_logprobs(x, None, None, None, pkg.DeviceArray(status, (1, 1), "int32"))
    with pytest.raises(RuntimeError, match="status 61"):
        cache.check()
    cache.check()
    k, at = _randn(_gen(1), 1, 70, 1, 64), _ints(70)
    cache.append(k, k, at)
    out = torch.empty(1, 1, 1, 64, device="cuda")
    cache.attention(k[:, :1], out, at)
    cache.check()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype,chain", [("f16", 64 * 16), ("bf16", 64 * 8)])
def test_sums_of_16_bit_portions_over_many_tokens(pkg, dtype, chain):
    """Weights of a few magnitudes over 32800 tokens of positive values: sums that lose up to a unit towards zero all lose it the same way."""
    g, t = _gen(109), TYPES[dtype]
    n, h, d, rows = 32800, 160, 32, 100
    k, v = torch.zeros(1, n, 1, d, device="cuda", dtype=t), (_randn(g, 1, n, 1, d).abs() + 0.5).to(t)
    k[..., 0] = torch.randint(-4, 5, (1, n, 1), generator=g, device="cuda").to(t)
    cache, at = _fill(pkg, k.expand(1, n, h, d), v.expand(1, n, h, d), n, [n])
    q = torch.zeros(1, rows, h, d, device="cuda", dtype=t)
    q[..., 0] = 0.3
    out = torch.full_like(q, 3.0)
    cache.attention(q, out, at, scale=1.0)
    cache.check()
    vv, s = plain.rounded(v)[0, :, 0], plain.rounded(k)[0, :, 0, 0] * q[0, 0, 0, 0].double()
    p = torch.exp(s)[:, None]
    want = ((p * vv).cumsum(0)[-rows:] / p.cumsum(0)[-rows:])[:, None]
    # a score is one product, exact, times a factor and against a reference (4 * 2^-24 of at most 1.2, twice in a weight); an exponential and terms
    # (2^-20; one term for bf16: 2^-12 each, either way); a sum in tensor memory loses up to 2^-23 with each of its `chain` products, less while it
    # is small: half of that on the whole; what is put aside is added up to nearest, (n / 128) times 2^-24 at most, and the result rounded
    terms = 2.0 ** -12 if dtype == "bf16" else 0.0
    limit = want * (2 * 1.2 * 4 * 2.0 ** -24 + 2.0 ** -20 + terms + chain * 2.0 ** -24 + n / 128 * 2.0 ** -24 + torch.finfo(t).eps / 2)
    err = (out[0].double() - want).abs()
    assert (err <= limit).all(), float((err / limit).max())


# ---------------------------------------------------------------------------------------------- around the borders between schemes

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs,rows,heads,kv_heads,dim,capacity", [
    (70, 1, 4, 2, 64, 1500), (33, 2, 8, 1, 128, 3000), (64, 1, 2, 2, 256, 700), (128, 1, 4, 1, 96, 2000),      # a few rows, sequences cut
    (70, 100, 2, 2, 64, 1500), (40, 120, 3, 3, 32, 2000),                                                       # many rows, cut
    (40, 1, 32, 8, 64, 500), (300, 1, 1, 1, 32, 400)])                                                          # a CTA a unit
def test_more_sequences_than_lanes(pkg, seqs, rows, heads, kv_heads, dim, capacity, dtype):
    """Sequences of very unequal lengths, some of no token, some shorter than their portion: every one has its place among the CTAs."""
    g, t = _gen(seqs + rows), TYPES[dtype]
    cuts = [0, 1, 31, 33, capacity, capacity // 7, capacity // 2 + 1, rows // 2, 129, capacity - 1]
    lengths = [min(capacity, cuts[(7 * i + i // 10) % len(cuts)]) for i in range(seqs)]
    real = [(rows, rows // 3, 0, rows)[i % 4] if rows > 1 else i % 9 != 4 for i in range(seqs)]
    real = [int(x) for x in real]
    k, v = (_randn(g, seqs, capacity, kv_heads, dim, dtype=t) for _ in range(2))
    cache, at = _fill(pkg, k, v, capacity, lengths)
    q = _randn(g, seqs, rows, heads, dim, dtype=t)
    mass = torch.full((seqs, kv_heads, capacity), -1.0, device="cuda")
    out, lse = torch.full_like(q, 3.0), torch.full((seqs, rows, heads), 4.0, device="cuda")
    for _ in range(3):                                                   # tickets and rooms are as they were each time
        cache.attention(q, out, at, rows=_ints(*real), lse=lse, mass_out=mass)
    cache.check()
    kk, vv = _held(k, None), _held(v, None)
    for i in range(seqs):
        n, m = lengths[i], real[i]
        assert (out[i, m:] == 3.0).all() and (lse[i, m:] == 4.0).all() and (mass[i, :, n:] == -1.0).all()
        empty = max(0, m - n)                                            # rows before token 0
        assert (out[i, :empty] == 0).all() and (lse[i, :empty] == -math.inf).all()
        if m == 0 or n == 0:
            assert (mass[i, :, :n] == 0).all()
            continue
        _check_by_component(out[i:i + 1, empty:], lse[i:i + 1, empty:], q[i:i + 1, empty:], kk[i, :, :n], vv[i, :, :n], m - empty, dim ** -0.5, t, mass[i:i + 1],
                            torch.zeros_like(mass[i:i + 1]))


@pytest.mark.parametrize("rows,heads,kv_heads,dim", [(1, 8, 2, 128), (16, 8, 2, 64), (5, 4, 1, 192), (150, 4, 2, 96)])
def test_a_cache_with_far_more_room_than_tokens(pkg, rows, heads, kv_heads, dim):
    """Rules on sizes see the room, kernels the lengths."""
    g, seqs, capacity, lengths = _gen(127), 3, 1 << 18, [1000, 150, 1]
    k, v = (_randn(g, seqs, 1000, kv_heads, dim) for _ in range(2))
    cache, at = _fill(pkg, k, v, capacity, lengths)
    q = _randn(g, seqs, rows, heads, dim)
    out, lse = torch.full_like(q, 3.0), torch.full((seqs, rows, heads), 4.0, device="cuda")
    mass = torch.full((seqs, kv_heads, capacity), -1.0, device="cuda")
    cache.attention(q, out, at, lse=lse, mass_out=mass)
    cache.check()
    kk, vv = _held(k, None), _held(v, None)
    for i, n in enumerate(lengths):
        empty = max(0, rows - n)
        assert (out[i, :empty] == 0).all() and (mass[i, :, n:] == -1.0).all()
        _check_by_component(out[i:i + 1, empty:], lse[i:i + 1, empty:], q[i:i + 1, empty:], kk[i, :, :n], vv[i, :, :n], rows - empty, dim ** -0.5, torch.float32, mass[i:i + 1],
                            torch.zeros_like(mass[i:i + 1]))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["random", "few values", "nan"])
def test_eviction_of_more_tokens_than_keys_are_held(pkg, kind, in_place):
    """Sequences on both sides of the 40960 tokens whose keys wait in shared memory."""
    g = _gen(131)
    lengths, keep, recent, first, h, d = [70001, 40960, 41003, 12000], 12345, 1000, 4, 2, 32
    s, capacity = len(lengths), 70001
    mass = torch.rand(s, h, capacity, generator=g, device="cuda")
    if kind == "few values":
        mass = (mass * 5).floor()
    elif kind == "nan":
        mass = torch.where(mass < 0.9, math.nan, mass)
    k = _randn(g, s, capacity, h, d, dtype=torch.bfloat16)
    cache, at = _fill(pkg, k, -k, capacity, lengths)
    into = cache if in_place else pkg.KV4Cache(s, h, d, keep)
    old, held = mass.clone(), plain.rounded(k)
    new_mass = mass if in_place else torch.full((s, h, keep), -1.0, device="cuda")
    new, kept = at if in_place else torch.empty_like(at), torch.full((s, h, keep), -7, dtype=torch.int32, device="cuda")
    cache.evict(into, at, new, mass, new_mass, kept, keep=keep, recent=recent, first=first)
    assert new.tolist() == [min(n, keep) for n in lengths]
    gk, gv = (torch.empty(s, keep, h, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    into.read(gk, gv, new, rows=new)
    for i, n in enumerate(lengths):
        for j in range(h):
            want = plain.kept(old[i, j], n, keep, recent, first)
            m = len(want)
            assert kept[i, j, :m].tolist() == want
            assert torch.equal(gk[i, :m, j].double(), held[i, want, j]) and torch.equal(gv[i, :m, j].double(), -held[i, want, j])
            a, b = new_mass[i, j, :m], old[i, j, want]
            assert torch.equal(torch.nan_to_num(a, nan=-2.0), torch.nan_to_num(b, nan=-2.0))
