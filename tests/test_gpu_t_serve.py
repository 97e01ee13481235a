"""The operators for servers of language models (include/voxtral_b200_serve.h) on the GPU, against the same in 64 bits."""
import math

import pytest
import torch

import serve_plain as plain

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DIMS = (32, 64, 96, 128, 192, 256)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _fill(pkg, k, v, capacity, lengths):
    """A cache that holds the first lengths[s] of k, v [seqs, n, H, D], through append."""
    s, n, h, d = k.shape
    cache = pkg.KV4Cache(s, h, d, capacity)
    at = _ints(*lengths)
    # token i of a sequence is row i of its portion: sequences end at different rows
    cache.append(k, v, at, rows=at)
    return cache, at


def _held(k, lengths):
    """What the cache stands for, [seqs, H, n, D] in 64 bits."""
    return plain.rounded(k).transpose(1, 2)


def _check_attention(got, lse, q, k, v, lengths, rows, scale, dtype, mass=None, mass_in=None):
    for s in range(q.shape[0]):
        n, t = lengths[s], rows[s]
        want, want_lse, want_mass = plain.attention(q[s], k[s], v[s], n, t, scale, None if mass_in is None else mass_in[s])
        score, result = plain.attention_bounds(q[s, :t], k[s][:, :n], v[s][:, :n], scale, dtype) if n and t else (1e-6, 1e-6)
        err = (got[s, :t].double() - want[:t]).abs()
        limit = result + torch.finfo(dtype).eps / 2 * want[:t].abs() + torch.finfo(dtype).tiny
        assert (err <= limit).all(), (s, float((err / limit).max()))
        if lse is not None:
            a, b = lse[s, :t].double(), want_lse[:t]
            assert torch.equal(torch.isinf(a), torch.isinf(b))
            fin = torch.isfinite(b)
            assert ((a - b).abs()[fin] <= score + 2.0 ** -22 * b.abs()[fin]).all(), (s, float((a - b).abs()[fin].max()), score)
        if mass is not None:
            m = mass[s, :, :n].double()
            lim = want_mass * (2 * score + 2.0 ** -20) + 1e-30
            assert ((m - want_mass).abs() <= lim).all(), (s, float(((m - want_mass).abs() / lim).max()))


# ---------------------------------------------------------------------------------------------- rows in and out

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_rows_are_rounded_as_the_format_says(pkg, dim, dtype):
    g = _gen(dim)
    t = TYPES[dtype]
    s, n, h = 3, 37, 3
    k, v = (_randn(g, s, n, h, dim) * torch.exp2(torch.randint(-12, 12, (s, n, h, 1), generator=g, device="cuda").float()) for _ in range(2))
    k[0, 0] = 0.0
    k[0, 1, 0, :32] = torch.tensor([0, .25, -.25, .75, -.75, 1.25, 1.75, 2.5, 3.5, 5, -5, 7, 7.9, 4, 6, -6] * 2, device="cuda")     # every tie, with the scale 1
    v[1, 2, 1, 5] = -0.0
    k, v = k.to(t), v.to(t)
    cache, at = _fill(pkg, k, v, 41, [n] * s)
    gk, gv = torch.full((s, n, h, dim), 9.0, device="cuda"), torch.full((s, n, h, dim), 9.0, device="cuda")
    cache.read(gk, gv, at)
    assert torch.equal(gk.double(), plain.rounded(k)) and torch.equal(gv.double(), plain.rounded(v))
    gk, gv = (torch.empty(s, n, h, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))      # two bits and a power of two: exact
    cache.read(gk, gv, at)
    assert torch.equal(gk.double(), plain.rounded(k)) and torch.equal(gv.double(), plain.rounded(v))


def test_values_that_are_not_finite_and_extremes(pkg):
    x = torch.zeros(1, 6, 1, 64, device="cuda")
    x[0, 0, 0, 3] = math.nan
    x[0, 1, 0, 40] = math.inf
    x[0, 2, 0, :] = torch.finfo(torch.float32).max
    x[0, 3, 0, :] = 2.0 ** -149
    x[0, 4, 0, :] = 2.0 ** -126
    x[0, 5, 0, :] = -1.5 * 2.0 ** -124
    cache, at = _fill(pkg, x, x, 6, [6])
    k, v = torch.empty_like(x), torch.empty_like(x)
    cache.read(k, v, at)
    want = plain.rounded(x)
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fin = ~torch.isnan(want)
        assert torch.equal(got.double()[fin], want[fin])


def test_ragged_portions_leave_the_rest_alone(pkg):
    g = _gen(5)
    s, h, d, cap = 5, 2, 64, 70
    cache = pkg.KV4Cache(s, h, d, cap)
    base = _randn(g, s, cap, h, d)
    cache.append(base, base, _ints(*[cap] * s))
    new = _randn(g, s, 9, h, d)
    lengths, rows = [9, 70, 33, 4, 80], [9, 3, 0, 7, 12]       # rows before token 0 and beyond the capacity: clipped
    cache.append(new, -new, _ints(*lengths), rows=_ints(*rows))
    want = plain.rounded(base).clone()
    for i in range(s):
        n, t = min(lengths[i], cap), min(rows[i], 9)
        for r in range(t):
            if n - t + r >= 0:
                want[i, n - t + r] = plain.rounded(new[i, r])
    k, v = torch.empty(s, cap, h, d, device="cuda"), torch.empty(s, cap, h, d, device="cuda")
    cache.read(k, v, _ints(*[cap] * s))
    assert torch.equal(k.double(), want)
    # reading a ragged portion leaves the rows beyond it as they are
    k.fill_(5.0)
    cache.read(k[:, :9], v[:, :9], _ints(*lengths), rows=_ints(*rows))
    for i in range(s):
        n, t = min(lengths[i], cap), min(rows[i], 9)
        for r in range(9):
            there = r < t and n - t + r >= 0
            assert torch.equal(k[i, r].double(), want[i, n - t + r] if there else torch.full((h, d), 5.0, device="cuda").double())
    assert (k[:, 9:] == 5.0).all()


@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (3, 5), (4, 8)])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(pkg, dtype, offset, pad):
    """q, k, v as parts of one packed projection, from any element on."""
    g = _gen(offset * 10 + pad)
    t = TYPES[dtype]
    s, n, h, heads, d = 2, 11, 2, 6, 64
    width = (heads + 2 * h) * d + pad
    x = _randn(g, s * n * width + offset, dtype=t)[offset:].view(s, n, width)
    q = x[..., :heads * d].unflatten(-1, (heads, d))
    k, v = (x[..., (heads + i * h) * d:(heads + (i + 1) * h) * d].unflatten(-1, (h, d)) for i in range(2))
    cache = pkg.KV4Cache(s, h, d, 16)
    at = _ints(n, n)
    cache.append(k, v, at)
    out = torch.full((s, heads, n, d), 7.0, device="cuda", dtype=t).transpose(1, 2)          # heads outside rows
    lse = torch.empty(s, n, heads, device="cuda")
    cache.attention(q, out, at, lse=lse)
    cache.check()
    _check_attention(out, lse, q, _held(k, None), _held(v, None), [n, n], [n, n], d ** -0.5, t)


# ---------------------------------------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_one_token(pkg, dim, dtype):
    g = _gen(dim + 1)
    t = TYPES[dtype]
    lengths = [1, 33, 300, 0, 32, 517]
    s, h, heads = len(lengths), 2, 8
    k, v = (_randn(g, s, max(lengths), h, dim, dtype=t) for _ in range(2))
    cache, at = _fill(pkg, k, v, max(lengths), lengths)
    q = _randn(g, s, 1, heads, dim, dtype=t)
    out, lse = torch.full_like(q, 3.0), torch.empty(s, 1, heads, device="cuda")
    mass_in = torch.rand(s, h, max(lengths), generator=g, device="cuda")
    mass = torch.full_like(mass_in, -1.0)
    cache.attention(q, out, at, lse=lse, mass_in=mass_in, mass_out=mass)
    cache.check()
    _check_attention(out, lse, q, _held(k, None), _held(v, None), lengths, [1] * s, dim ** -0.5, t, mass, mass_in)
    for i, n in enumerate(lengths):
        assert (mass[i, :, n:] == -1.0).all()                  # behind a sequence: as it was


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,rows,lengths", [
    (8, 8, 64, [1, 1], [40, 3]), (6, 2, 128, [5, 2], [5, 700]), (12, 2, 96, [3, 0], [129, 64]), (7, 1, 32, [4, 4], [2, 65]),
    (64, 8, 128, [2, 1], [1000, 31]), (4, 1, 256, [9, 7], [300, 9]), (5, 5, 192, [17, 13], [600, 20]), (40, 2, 64, [33, 1], [257, 1])])
def test_a_few_rows(pkg, heads, kv_heads, dim, rows, lengths, dtype):
    g = _gen(heads * dim)
    t = TYPES[dtype]
    s, n, m = len(rows), max(lengths), max(rows)
    k, v = (_randn(g, s, n, kv_heads, dim, dtype=t) for _ in range(2))
    cache, at = _fill(pkg, k, v, n + 3, lengths)
    q = _randn(g, s, m, heads, dim, dtype=t)
    out, lse = torch.full_like(q, 3.0), torch.full((s, m, heads), 4.0, device="cuda")
    mass = torch.full((s, kv_heads, n + 3), -1.0, device="cuda")
    cache.attention(q, out, at, rows=_ints(*rows), lse=lse, mass_out=mass)
    cache.check()
    _check_attention(out, lse, q, _held(k, None), _held(v, None), lengths, rows, dim ** -0.5, t, mass)
    for i in range(s):
        assert (out[i, rows[i]:] == 3.0).all() and (lse[i, rows[i]:] == 4.0).all() and (mass[i, :, lengths[i]:] == -1.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,rows,length", [(8, 2, 128, 150, 150), (8, 8, 64, 65, 400), (4, 2, 96, 130, 190), (6, 2, 192, 70, 333), (2, 1, 256, 90, 100),
                                                          (16, 1, 32, 64, 77), (5, 1, 128, 257, 1025), (32, 32, 64, 129, 200), (4, 2, 128, 100, 1500), (4, 4, 96, 66, 900), (32, 32, 32, 129, 2100), (27, 27, 32, 129, 2100)])
def test_portions_of_a_prompt(pkg, heads, kv_heads, dim, rows, length, dtype):
    g = _gen(rows * dim)
    t = TYPES[dtype]
    lengths, real = [length, rows + 1, rows // 2], [rows, rows - 1, rows // 2]
    s = len(lengths)
    k, v = (_randn(g, s, max(lengths), kv_heads, dim, dtype=t) for _ in range(2))
    cache, at = _fill(pkg, k, v, max(lengths), lengths)
    q = _randn(g, s, rows, heads, dim, dtype=t)
    out, lse = torch.full_like(q, 3.0), torch.full((s, rows, heads), 4.0, device="cuda")
    mass_in = torch.rand(s, kv_heads, max(lengths), generator=g, device="cuda")
    mass = torch.full_like(mass_in, -1.0)
    cache.attention(q, out, at, rows=_ints(*real), lse=lse, mass_in=mass_in, mass_out=mass)
    cache.check()
    _check_attention(out, lse, q, _held(k, None), _held(v, None), lengths, real, dim ** -0.5, t, mass, mass_in)
    for i in range(s):
        assert (out[i, real[i]:] == 3.0).all() and (lse[i, real[i]:] == 4.0).all() and (mass[i, :, lengths[i]:] == -1.0).all()


@pytest.mark.parametrize("rows", [1, 100])
@pytest.mark.parametrize("scale", [3.0, -0.5, 0.0])
def test_sharp_and_flat_weights(pkg, scale, rows):
    g = _gen(17)
    s, n, h, heads, d = 1, 400, 1, 4, 64
    k, v = _randn(g, s, n, h, d) * 3.0, _randn(g, s, n, h, d)
    cache, at = _fill(pkg, k, v, n, [n])
    q = _randn(g, s, rows, heads, d)
    out, lse = torch.empty_like(q), torch.empty(s, rows, heads, device="cuda")
    cache.attention(q, out, at, scale=scale, lse=lse)
    _check_attention(out, lse, q, _held(k, None), _held(v, None), [n], [rows], scale, torch.float32)


@pytest.mark.parametrize("rows", [1, 80])
def test_values_of_very_different_magnitude(pkg, rows):
    """Value scales from 2^-60 to 2^60 in one cache, the large ones at tokens that weigh nothing, and the other way round."""
    g = _gen(23)
    n, h, heads, d = 200, 1, 2, 128
    k, q = _randn(g, 1, n, h, d), _randn(g, 1, rows, heads, d)
    v = _randn(g, 1, n, h, d) * torch.exp2(torch.randint(-60, 60, (1, n, h, 1), generator=g, device="cuda").float())
    cache, at = _fill(pkg, k, v, n, [n])
    out, lse = torch.empty_like(q), torch.empty(1, rows, heads, device="cuda")
    cache.attention(q, out, at, lse=lse)
    _check_attention(out, lse, q, _held(k, None), _held(v, None), [n], [rows], d ** -0.5, torch.float32)
    # keys over 40 binary orders: a score counts by its own magnitude
    k = _randn(g, 1, n, h, d) * torch.exp2(torch.randint(-40, 1, (1, n, h, 1), generator=g, device="cuda").float())
    cache, at = _fill(pkg, k, _randn(g, 1, n, h, d), n, [n])
    kk, vv = torch.empty(1, n, h, d, device="cuda"), torch.empty(1, n, h, d, device="cuda")
    cache.read(kk, vv, at)
    cache.attention(q, out, at, lse=lse)
    _check_attention(out, lse, q, kk.transpose(1, 2), vv.transpose(1, 2), [n], [rows], d ** -0.5, torch.float32)


@pytest.mark.parametrize("dtype,n,rise,fall", [("f32", 7001, 0, 20), ("f32", 7001, 20, 20), ("f32", 7001, 80, 20), ("f16", 33001, 4, 4), ("bf16", 33001, 20, 20)])
def test_many_rows_over_many_tokens(pkg, dtype, n, rise, fall):
    """More units than SMs and far more tokens than a sum stays in one place. Halfway the scores rise by `rise` binary orders while values
    fall by `fall`: both halves count where the two are alike."""
    g = _gen(61)
    h, d, rows, half, t = 160, 32, 100, n // 2, TYPES[dtype]
    k, v = torch.zeros(1, n, h, d, device="cuda", dtype=t), _randn(g, 1, n, h, d, dtype=t).abs()
    k[:, half:, :, 0] = 4.0
    v[:, :half] *= 2.0 ** fall
    cache, at = _fill(pkg, k, v, n, [n])
    q = _randn(g, 1, rows, h, d, dtype=t) * 0.0
    q[..., 0] = rise * math.log(2.0) / 4.0
    out, lse = torch.full_like(q, 3.0), torch.full((1, rows, h), 4.0, device="cuda")
    cache.attention(q, out, at, scale=1.0, lse=lse)
    cache.check()
    vv = _held(v, None)[0]                                               # [h, n, d]
    seen = [half, n - rows - half + 1]                                   # of each half by the first row, one more of the second a row
    early, late = vv[:, :half].sum(1), vv[:, half:].cumsum(1)[:, -rows:].transpose(0, 1)
    rise_exact = float(q[0, 0, 0, 0].double()) * 4.0                     # natural
    w = math.exp(-rise_exact)
    count = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None, None] + seen[1]
    want = (early[None] * w + late) / (half * w + count)
    # a score: queries as two terms, products and factors; a weight: twice that, exponentials and terms (2^-20), and FP16's smallest step of its
    # second term, 2^-32 of the largest weight, for every early token (one term for bf16: 2^-11, normal numbers here); sums: a unit for each 16
    # tokens and term, and the scales' factors; the result's own rounding
    score = rise_exact * (2.0 ** -22 + 10 * 2.0 ** -23)
    limit = want * (2 * score + 2.0 ** -19 + (n / 8 + 16) * 2.0 ** -23 + (2.0 ** -11 if dtype == "bf16" else 0.0) + torch.finfo(t).eps / 2) + early[None] * 2.0 ** -32 / count
    assert ((out[0].double() - want).abs() <= limit).all()
    total = torch.log(half * w + count[..., 0]) + rise_exact
    assert ((lse[0].double() - total).abs() <= score + 2.0 ** -18 + total.abs() * 2.0 ** -23).all()


@pytest.mark.parametrize("rows", [3, 90])
def test_what_a_row_does_not_see_does_not_reach_it(pkg, rows):
    """NaN and infinities in later tokens, and in what an earlier sequence has left behind the last one."""
    g = _gen(29)
    n, h, heads, d = 150, 1, 2, 128
    k, v = _randn(g, 1, n, h, d), _randn(g, 1, n, h, d)
    dirty = torch.full((1, n, h, d), math.nan, device="cuda")
    cache = pkg.KV4Cache(1, h, d, n)
    cache.append(dirty, dirty, _ints(n))
    length = n - 20
    k2, v2 = k.clone(), v.clone()
    k2[0, length - 1], v2[0, length - 1, 0, 7] = math.nan, math.inf               # the last row's own token
    cache.append(k2, v2, _ints(length), rows=_ints(length))
    q = _randn(g, 1, rows, heads, d)
    out, lse = torch.empty_like(q), torch.empty(1, rows, heads, device="cuda")
    cache.attention(q, out, _ints(length), lse=lse)
    _check_attention(out, lse, q[:, :rows - 1], _held(k, None)[:, :, :length - 1], _held(v, None)[:, :, :length - 1], [length - 1], [rows - 1], d ** -0.5, torch.float32)
    assert torch.isnan(out[0, rows - 1]).all() and torch.isnan(lse[0, rows - 1]).all()
    # a value that is not finite in a token that is seen: its block of 32, no other
    k2[0, length - 1] = k[0, length - 1]
    cache.append(k2, v2, _ints(length), rows=_ints(length))
    cache.attention(q, out, _ints(length), lse=lse)
    assert torch.isnan(out[0, rows - 1, :, :32]).all() and torch.isfinite(out[0, rows - 1, :, 32:]).all() and torch.isfinite(out[0, :rows - 1]).all()


def test_offsets_beyond_32_bits(pkg):
    """The last head of a cache of 9 GB: its rows lie beyond 2^32 bytes, its tokens beyond 2^32 / 8 elements."""
    g = _gen(31)
    s, h, d, cap = 4, 16, 128, 1 << 20
    cache = pkg.KV4Cache(s, h, d, cap)
    n = 300
    k, v = _randn(g, s, n, h, d, dtype=torch.bfloat16), _randn(g, s, n, h, d, dtype=torch.bfloat16)
    # the portion is tokens cap - n .. of the last sequence; everything before it is zeros, which the scores know
    at, rows = _ints(0, 0, 0, cap), _ints(0, 0, 0, n)
    cache.append(k, v, at, rows=rows)
    q = _randn(g, s, 1, h, d, dtype=torch.bfloat16) * 4.0
    out, lse = torch.zeros_like(q), torch.empty(s, 1, h, device="cuda")
    mass = torch.zeros(s, h, cap, device="cuda")
    cache.attention(q, out, at, lse=lse, mass_out=mass)
    cache.check()
    kk, vv = _held(k, None)[3], _held(v, None)[3]
    x = torch.einsum("hd,hnd->hn", q[3, 0].double(), kk) * d ** -0.5
    z = torch.logsumexp(torch.cat((x, torch.full((h, 1), math.log(cap - n), device="cuda", dtype=torch.float64)), 1), 1)
    p = torch.exp(x - z[:, None])
    want = torch.einsum("hn,hnd->hd", p, vv)
    score, _ = plain.attention_bounds(q[3], kk, vv, d ** -0.5, torch.bfloat16)
    # every weight within a score's error twice and a term's rounding; the other tokens are zeros
    limit = float(vv.abs().amax()) * p.sum(1, keepdim=True) * (2 * score + 2.0 ** -11 + (cap / 16) * 2.0 ** -23) + want.abs() * 2.0 ** -8 + 1e-7
    assert ((out[3, 0].double() - want).abs() <= limit).all()
    assert ((mass[3, :, cap - n:].double() - p).abs() <= p * (2 * score + 2.0 ** -18)).all()
    assert (out[:3] == 0).all() and (mass[:3] == 0).all()


def test_same_bits_every_time(pkg):
    g = _gen(37)
    s, n, h, heads, d = 2, 3000, 2, 16, 128
    k, v = _randn(g, s, n, h, d), _randn(g, s, n, h, d)
    cache, at = _fill(pkg, k, v, n, [n, n - 100])
    q = _randn(g, s, 2, heads, d)
    first = None
    for _ in range(20):
        out, lse, mass = torch.empty_like(q), torch.empty(s, 2, heads, device="cuda"), torch.zeros(s, h, n, device="cuda")
        cache.attention(q, out, at, lse=lse, mass_out=mass)
        got = (out, lse, mass)
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


# ---------------------------------------------------------------------------------------------- eviction

def _check_eviction(pkg, lengths, keep, recent, first, mass, dim=64, in_place=False, alias=False):
    g = _gen(41)
    s, h, cap = mass.shape
    k, v = _randn(g, s, cap, h, dim), _randn(g, s, cap, h, dim)
    cache, at = _fill(pkg, k, v, cap, lengths)
    into = cache if in_place else pkg.KV4Cache(s, h, dim, keep + 3)
    kept = torch.full((s, h, keep), -7, dtype=torch.int32, device="cuda")
    old = mass.clone()
    new_mass = mass if alias else torch.full((s, h, keep), -1.0, device="cuda")
    new = at if alias else torch.empty_like(at)
    cache.evict(into, at, new, mass, new_mass, kept, keep=keep, recent=recent, first=first)
    size = into.capacity
    gk, gv = torch.empty(s, size, h, dim, device="cuda"), torch.empty(s, size, h, dim, device="cuda")
    into.read(gk, gv, _ints(*[size] * s))
    hk, hv = plain.rounded(k), plain.rounded(v)
    for i, n in enumerate(lengths):
        assert int(new[i]) == min(n, keep)
        for j in range(h):
            want = plain.kept(old[i, j], n, keep, recent, first)
            m = len(want)
            assert kept[i, j, :m].tolist() == want, (i, j)
            assert (kept[i, j, m:] == -7).all()
            assert torch.equal(gk[i, :m, j].double(), hk[i, want, j]) and torch.equal(gv[i, :m, j].double(), hv[i, want, j])
            a, b = new_mass[i, j, :m], old[i, j, want]
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~torch.isnan(a)], b[~torch.isnan(b)])
            if not alias:
                assert (new_mass[i, j, m:] == -1.0).all()
            if in_place and n < cap:         # behind the last token: as it was
                assert torch.equal(gk[i, n:, j].double(), torch.zeros_like(hk[i, n:, j]))
            if not in_place:
                assert (gk[i, m:, j] == 0).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lengths,keep,recent,first", [
    ([100, 7, 0, 64], 64, 16, 4), ([1500, 1025, 1024, 1], 1024, 100, 0), ([2000, 33, 31, 32], 32, 0, 0), ([50, 2, 1, 3], 1, 0, 0), ([90, 80, 70, 60], 60, 59, 1),
    ([40, 10, 1999, 500], 2000, 5, 5), ([700, 701, 702, 703], 5, 3, 1)])
def test_eviction(pkg, lengths, keep, recent, first, in_place):
    g = _gen(keep)
    mass = torch.rand(len(lengths), 3, 2000, generator=g, device="cuda")
    _check_eviction(pkg, lengths, keep, recent, first, mass, in_place=in_place)


@pytest.mark.parametrize("dim", DIMS)
def test_eviction_of_every_row_size(pkg, dim):
    mass = torch.rand(2, 2, 500, generator=_gen(dim), device="cuda")
    _check_eviction(pkg, [500, 299], 300, 20, 4, mass, dim=dim)
    _check_eviction(pkg, [500, 299], 300, 20, 4, mass, dim=dim, in_place=True, alias=True)


def test_eviction_in_place_of_more_heads_than_run_at_once(pkg):
    """The new lengths over the old ones: the heads that come last find the new ones there."""
    mass = torch.rand(2, 1100, 60, generator=_gen(71), device="cuda")
    _check_eviction(pkg, [60, 57], 40, 8, 2, mass, dim=32, in_place=True, alias=True)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "nan", "negative", "infinite", "tiny"])
def test_eviction_where_masses_tie_or_are_no_numbers(pkg, kind):
    g = _gen(7)
    mass = torch.rand(2, 2, 900, generator=g, device="cuda")
    if kind == "equal":
        mass.fill_(0.25)
    elif kind == "zeros":
        mass = torch.where(mass < 0.5, 0.0, -0.0)
    elif kind == "few values":
        mass = (mass * 3).floor()
    elif kind == "nan":
        mass = torch.where(mass < 0.7, math.nan, mass)
    elif kind == "negative":
        mass -= 0.5
    elif kind == "infinite":
        mass = torch.where(mass < 0.2, math.inf, torch.where(mass > 0.8, -math.inf, mass))
    else:
        mass *= 1e-41
    _check_eviction(pkg, [900, 333], 300, 10, 2, mass)


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_sequence_served_with_eviction(pkg, dtype):
    """Prompt, tokens, eviction in place, tokens again: every attention against 64 bits over the same cache."""
    g = _gen(53)
    t = TYPES[dtype]
    s, h, heads, d, cap, keep = 2, 2, 8, 128, 96, 64
    cache = pkg.KV4Cache(s, h, d, cap)
    mass = torch.zeros(s, h, cap, device="cuda")
    kept = torch.empty(s, h, keep, dtype=torch.int32, device="cuda")
    held = [[torch.zeros(h, 0, d, device="cuda", dtype=torch.float64) for _ in range(s)] for _ in range(2)]
    at = _ints(0, 0)

    def portion(rows):
        nonlocal at
        k, v, q = _randn(g, s, rows, h, d, dtype=t), _randn(g, s, rows, h, d, dtype=t), _randn(g, s, rows, heads, d, dtype=t)
        at += rows
        before = mass.clone()
        cache.append(k, v, at)
        out, lse = torch.empty_like(q), torch.empty(s, rows, heads, device="cuda")
        cache.attention(q, out, at, lse=lse, mass_in=mass, mass_out=mass)
        for x, new in zip(held, (k, v)):
            for i in range(s):
                x[i] = torch.cat((x[i], plain.rounded(new[i]).transpose(0, 1)), 1)
        lengths = at.tolist()
        _check_attention(out, lse, q, held[0], held[1], lengths, [rows] * s, d ** -0.5, t, mass, before)

    portion(80)
    for _ in range(3):
        portion(1)
    for _ in range(2):
        before = mass.clone()
        n = at.tolist()
        cache.evict(cache, at, at, mass, mass, kept, keep=keep, recent=8, first=2)
        for i in range(s):
            want = [plain.kept(before[i, j], n[i], keep, 8, 2) for j in range(h)]
            assert kept[i].tolist() == want
            for x in held:
                x[i] = torch.stack([x[i][j, want[j]] for j in range(h)])
        assert at.tolist() == [keep] * s
        for _ in range(4):
            portion(1)
        portion(3)
    cache.check()


def test_captured_and_replayed(pkg):
    """A token's calls in a graph, replayed with new inputs in the same arrays; two graphs of one cache in turn, on another stream."""
    g = _gen(59)
    s, h, heads, d, cap = 2, 2, 8, 128, 2000
    cache = pkg.KV4Cache(s, h, d, cap)
    k, v, q = _randn(g, s, 1, h, d), _randn(g, s, 1, h, d), _randn(g, s, 1, heads, d)
    out, lse, mass = torch.empty_like(q), torch.empty(s, 1, heads, device="cuda"), torch.zeros(s, h, cap, device="cuda")
    x = _randn(g, s, 1000)
    tokens, lp = _ints(3, 999), torch.empty(s, device="cuda")
    at, one = _ints(1500, 20), _ints(1, 1)
    base = _randn(g, s, cap, h, d)
    cache.append(base, base, _ints(cap, cap))
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            st = torch.cuda.current_stream().cuda_stream
            at += one
            cache.append(k, v, at, stream=st)
            cache.attention(q, out, at, lse=lse, mass_out=mass, stream=st)
            pkg.token_logprobs(x, tokens, lp, stream=st)
        graphs.append(graph)
    held = [plain.rounded(base).clone() for _ in range(2)]
    n = [1500, 20]
    for i in range(6):
        k.copy_(_randn(g, s, 1, h, d))
        q.copy_(_randn(g, s, 1, heads, d))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[i % 2].replay()
        torch.cuda.synchronize()
        n = [a + 1 for a in n]
        assert at.tolist() == n
        for j in range(s):
            held[0][j, n[j] - 1] = plain.rounded(k[j, 0])
            held[1][j, n[j] - 1] = plain.rounded(v[j, 0])
        _check_attention(out, lse, q, held[0].transpose(1, 2), held[1].transpose(1, 2), n, [1, 1], d ** -0.5, torch.float32, mass)
    assert torch.allclose(lp.double().cpu(), plain.logprobs(x, tokens, 0)[0], atol=1e-5)


def test_portions_captured_and_replayed_side_by_side(pkg):
    """Portions of many rows of two caches, in graphs on two streams at once, replayed with new lengths and queries: every time the bits of the
    calls by themselves, which are right; the masses go on from what they were."""
    g = _gen(67)
    s, h, heads, d, cap, rows = 2, 4, 16, 128, 3000, 200
    lengths = [[3000, 700], [200, 2999], [1500, 2200]]
    base, v0 = _randn(g, s, cap, h, d), _randn(g, s, cap, h, d)
    qs = [_randn(g, s, rows, heads, d) for _ in lengths]
    kh, vh = _held(base, None), _held(v0, None)
    alone, _ = _fill(pkg, base, v0, cap, [cap, cap])
    want = []
    for n, q in zip(lengths, qs):
        out, lse, mass = torch.empty_like(q), torch.empty(s, rows, heads, device="cuda"), torch.ones(s, h, cap, device="cuda")
        alone.attention(q, out, _ints(*n), lse=lse, mass_in=mass, mass_out=mass)
        _check_attention(out, lse, q, kh, vh, n, [rows, rows], d ** -0.5, torch.float32, mass, torch.ones(s, h, cap, device="cuda"))
        want.append((out, lse, mass))
    sides = []
    for _ in range(2):
        cache, at = _fill(pkg, base, v0, cap, [cap, cap])
        st, graph, q = torch.cuda.Stream(), torch.cuda.CUDAGraph(), qs[0].clone()
        got = (torch.empty_like(q), torch.empty(s, rows, heads, device="cuda"), torch.ones(s, h, cap, device="cuda"))
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            cache.attention(q, got[0], at, lse=got[1], mass_in=got[2], mass_out=got[2], stream=torch.cuda.current_stream().cuda_stream)
        sides.append((cache, at, q, got, st, graph))
    for i in range(6):
        for _, at, q, got, _, _ in sides:
            at.copy_(_ints(*lengths[i % 3]))
            q.copy_(qs[i % 3])
            got[2].fill_(1.0)
        torch.cuda.synchronize()
        for *_, st, graph in sides:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for cache, _, _, got, _, _ in sides:
            cache.check()
            assert all(torch.equal(x, y) for x, y in zip(got, want[i % 3]))


def test_two_caches_at_once(pkg):
    """Attention of two caches on two streams side by side, many times: workspaces are a cache's own."""
    g = _gen(61)
    s, n, h, heads, d = 1, 4000, 2, 8, 128
    made = []
    for i in range(2):
        k, v = _randn(g, s, n, h, d), _randn(g, s, n, h, d)
        cache, at = _fill(pkg, k, v, n, [n])
        q = _randn(g, s, 1, heads, d)
        alone, lse = torch.empty_like(q), torch.empty(s, 1, heads, device="cuda")
        cache.attention(q, alone, at, lse=lse)
        made.append((cache, at, q, alone, lse, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[torch.empty_like(m[3]) for _ in range(50)] for m in made]
    for i in range(50):
        for (cache, at, q, _, lse, st), o in zip(made, outs):
            cache.attention(q, o[i], at, lse=lse, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for m, o in zip(made, outs):
        assert all(torch.equal(x, m[3]) for x in o)


# ---------------------------------------------------------------------------------------------- what is refused, and nothing at all

def test_portions_of_no_rows(pkg):
    s, h, d, n = 2, 2, 64, 40
    k = _randn(_gen(1), s, n, h, d)
    cache, at = _fill(pkg, k, k, n, [n, 7])
    none = torch.empty(s, 0, h, d, device="cuda")
    cache.append(none, none, at)
    cache.read(none, none, at)
    q, lse = torch.empty(s, 0, 4, d, device="cuda"), torch.empty(s, 0, 4, device="cuda")
    cache.attention(q, q, at)
    mass_in, mass = torch.rand(s, h, n, device="cuda"), torch.full((s, h, n), -1.0, device="cuda")
    cache.attention(q, q, at, lse=lse, mass_in=mass_in, mass_out=mass)
    assert torch.equal(mass[0], mass_in[0]) and torch.equal(mass[1, :, :7], mass_in[1, :, :7]) and (mass[1, :, 7:] == -1.0).all()
    # rows there are, of which none is real
    q, lse = torch.randn(s, 3, 4, d, device="cuda"), torch.full((s, 3, 4), 5.0, device="cuda")
    out = torch.full_like(q, 5.0)
    cache.attention(q, out, at, rows=_ints(0, 0), lse=lse, mass_in=mass_in, mass_out=mass)
    assert (out == 5.0).all() and (lse == 5.0).all() and torch.equal(mass[0], mass_in[0])
    cache.check()


def test_calls_that_are_refused(pkg):
    import ctypes as C
    import sys
    serve = sys.modules[pkg.__name__ + ".serve"]
    L = serve.serve_lib()
    cache, small = pkg.KV4Cache(2, 2, 64, 32), pkg.KV4Cache(2, 2, 64, 8)
    k, at, q = torch.zeros(2, 3, 2, 64, device="cuda"), _ints(3, 3), torch.zeros(2, 3, 4, 64, device="cuda")
    host = torch.zeros(2, 3, 2, 64)
    p = lambda t: t.data_ptr()  # noqa: E731

    def refused(fn, handles, args, word):
        assert fn(*handles, C.byref(args), None) == -1
        assert word in L.vb200_serve_error().decode(), L.vb200_serve_error()

    rows = lambda t, kind=0: serve._Rows(p(t), kind, 384, 128, 64)  # noqa: E731
    for args, word in ((serve._AppendArgs(None, None, 3, rows(k), rows(k)), "needed"), (serve._AppendArgs(p(at), None, -1, rows(k), rows(k)), "negative"),
                       (serve._AppendArgs(p(at), None, 3, rows(k), rows(k, 1)), "one type"), (serve._AppendArgs(p(at), None, 3, rows(k, 7), rows(k, 7)), "one type"),
                       (serve._AppendArgs(p(at), None, 3, rows(host), rows(host)), "does not lie"),
                       (serve._AppendArgs(p(at), None, 3, serve._Rows(p(k) + 2, 0, 384, 128, 64), rows(k)), "aligned")):
        refused(L.vb200_kv4_append, (cache.h,), args, word)
        refused(L.vb200_kv4_read, (cache.h,), args, word)
    att = dict(lengths=p(at), rows=None, max_rows=3, heads=4, scale=1.0, q=rows(q), out=rows(q), lse=None, mass_in=None, mass_out=None)
    for change, word in (({"heads": 3}, "multiple"), ({"heads": 0}, "multiple"), ({"q": rows(q, 1)}, "one type"), ({"lengths": None}, "needed"), ({"max_rows": -2}, "negative"),
                         ({"mass_out": p(k)}, "lse"), ({"mass_in": p(k)}, "without"), ({"scale": math.nan}, "finite"), ({"scale": math.inf}, "finite"),
                         ({"q": rows(host), "out": rows(host)}, "does not lie"), ({"max_rows": 1 << 30, "heads": 8}, "too many")):
        refused(L.vb200_kv4_attention, (cache.h,), serve._AttentionArgs(**dict(att, **change)), word)
    mass, kept = torch.zeros(2, 2, 32, device="cuda"), torch.zeros(2, 2, 8, dtype=torch.int32, device="cuda")
    ev = dict(lengths=p(at), new_lengths=p(at), mass=p(mass), new_mass=p(mass), new_mass_ld=32, kept=p(kept), keep=8, recent=2, first=1)
    for change, word in (({"keep": 0}, "keep"), ({"recent": 8}, "together"), ({"first": -1}, "not negative"), ({"new_mass_ld": 7}, "new_mass_ld"), ({"kept": None}, "needed"),
                         ({"new_mass_ld": 31}, "may be mass")):
        refused(L.vb200_kv4_evict, (cache.h, cache.h), serve._EvictArgs(**dict(ev, **change)), word)
    refused(L.vb200_kv4_evict, (cache.h, small.h), serve._EvictArgs(**dict(ev, keep=9)), "more than into")
    refused(L.vb200_kv4_evict, (cache.h, small.h), serve._EvictArgs(**ev), "may be mass")
    refused(L.vb200_kv4_evict, (cache.h, pkg.KV4Cache(2, 1, 64, 8).h), serve._EvictArgs(**ev), "other seqs")
    call = cache.append_call(k, k, at)
    call()
    cache.close()
    with pytest.raises(ValueError, match="closed"):
        call()
    x = torch.zeros(2, 5)
    refused(L.vb200_token_logprobs, (), serve._LogprobsArgs(p(x), 0, 2, 5, 5, p(at), p(k), None, 0, None, None), "do not lie")


def test_first_call_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    code = """
import sys
sys.path.insert(0, %r)
import conftest, torch
pkg = conftest.load_package()
cache = pkg.KV4Cache(1, 1, 64, 100)
k, q = torch.randn(1, 70, 1, 64, device="cuda"), torch.randn(1, 70, 2, 64, device="cuda")
at, kept = torch.tensor([70], dtype=torch.int32, device="cuda"), torch.empty(1, 1, 20, dtype=torch.int32, device="cuda")
new = torch.empty_like(at)
out, lse, mass = torch.empty_like(q), torch.empty(1, 70, 2, device="cuda"), torch.zeros(1, 1, 100, device="cuda")
x, tok, lp = torch.randn(3, 5000, device="cuda"), torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(graph, stream=side):
    st = torch.cuda.current_stream().cuda_stream
    pkg.token_logprobs(x, tok, lp, stream=st)
    cache.append(k, k, at, stream=st)
    cache.attention(q, out, at, lse=lse, mass_out=mass, stream=st)
    cache.attention(q[:, :1], out[:, :1], at, stream=st)
    cache.evict(cache, at, new, mass, mass, kept, keep=20, stream=st)
graph.replay()
torch.cuda.synchronize()
cache.check()
assert torch.allclose(lp, torch.log_softmax(x, -1)[torch.arange(3), tok.long()], atol=1e-5)
assert int(new) == 20 and abs(float(lse.exp().isfinite().all()) - 1) == 0
print("OK")
""" % os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "OK" in r.stdout, (r.stdout[-2000:], r.stderr[-3000:])


# ---------------------------------------------------------------------------------------------- log probabilities

def _check_logprobs(pkg, x, tokens, top):
    rows = x.shape[0]
    lp, ent = torch.full((rows,), 5.0, device="cuda"), torch.full((rows,), 5.0, device="cuda")
    ids, tops = (torch.full((rows, top), -5, dtype=torch.int32, device="cuda"), torch.full((rows, top), 5.0, device="cuda")) if top else (None, None)
    pkg.token_logprobs(x, tokens, lp, ent, ids, tops)
    torch.cuda.synchronize()
    want_lp, want_ent, want_ids, want_tops = plain.logprobs(x, tokens, top)

    def near(got, want, what):
        got = got.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), what
        assert torch.equal(got == -math.inf, want == -math.inf), what
        fin = torch.isfinite(want)
        # a value's difference from the maximum, and the logarithm, at 2^-24; the sum: a thread's 2^-24 a value, at most 512 of them,
        # exponentials 2^-21 and 2^-23 of the argument, which counts with its weight (|x - m| e^(x - m) < 0.37)
        limit = 2.0 ** -22 * want[fin].abs() + 512 * 2.0 ** -24 + 2.0 ** -20
        assert ((got - want)[fin].abs() <= limit).all(), (what, float((got - want)[fin].abs().max()))

    near(lp, want_lp, "logprobs")
    # the entropy sums p (x - m): its terms by the same roundings, of sum p |x - m| <= log(vocab) + 1
    got, fin = ent.double().cpu(), torch.isfinite(want_ent)
    assert torch.equal(torch.isnan(got), torch.isnan(want_ent))
    assert ((got - want_ent)[fin].abs() <= (512 * 2.0 ** -24 + 2.0 ** -19) * (math.log(x.shape[1]) + 2)).all()
    if top:
        assert torch.equal(ids.cpu().long(), want_ids)
        near(tops, want_tops, "top")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 100, 32), (1, 1000, 0), (4, 1025, 20), (2, 4099, 32), (70, 8191, 5), (1, 131072, 32),
                                            (3, 262147, 7), (300, 513, 1), (40, 32768, 20)])
def test_logprobs(pkg, rows, vocab, top, dtype):
    g = _gen(vocab)
    x = (_randn(g, rows, vocab) * 3.0).to(TYPES[dtype])
    _check_logprobs(pkg, x, torch.randint(vocab, (rows,), generator=g, device="cuda").int(), top)


@pytest.mark.parametrize("offset,pad", [(1, 0), (3, 5), (7, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_of_rows_anywhere(pkg, dtype, offset, pad):
    g = _gen(offset)
    rows, vocab = 9, 5003
    x = (_randn(g, rows * (vocab + pad) + offset) * 2.0).to(TYPES[dtype])[offset:].view(rows, vocab + pad)[:, :vocab]
    _check_logprobs(pkg, x, torch.randint(vocab, (rows,), generator=g, device="cuda").int(), 20)


@pytest.mark.parametrize("vocab", [777, 50021])
def test_logprobs_of_masked_and_strange_rows(pkg, vocab):
    g = _gen(3)
    x = _randn(g, 12, vocab) * 2.0
    tokens = torch.randint(vocab, (12,), generator=g, device="cuda").int()
    x[0] = -math.inf                                       # nothing is left
    x[1] = -math.inf
    x[1, vocab // 2] = -3.0                                # one is
    x[2, ::2] = -math.inf
    x[3, 5] = math.nan
    x[4, vocab - 1] = math.inf
    x[5] = 1.25                                            # all tie
    x[6] = torch.arange(vocab, device="cuda") * 1e-3       # rising: every value is a new largest
    x[7] = -torch.arange(vocab, device="cuda") * 1e-3
    x[8] = torch.where(x[8] > 0, 0.0, -0.0)                # zeros of both signs tie
    x[9] = torch.finfo(torch.float32).min                  # a mask's lowest value
    x[9, 3] = 1.0
    x[10] = torch.finfo(torch.float32).min
    tokens[1], tokens[2], tokens[9] = vocab // 2, 0, 4
    tokens[7], tokens[11] = -1, vocab
    _check_logprobs(pkg, x, tokens, 32)
    x[6] = torch.arange(vocab, device="cuda").flip(0) // 7
    _check_logprobs(pkg, x, tokens, 9)
    _check_logprobs(pkg, x[:1].expand(4, vocab), tokens[:4], 3)      # rows of stride 0


def test_logprobs_one_output_at_a_time(pkg):
    g = _gen(9)
    x = _randn(g, 3, 3000)
    tokens = _ints(1, 2, 3)
    want = plain.logprobs(x, tokens, 4)
    lp, ent, tops = torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty(3, 4, device="cuda")
    ids = torch.empty(3, 4, dtype=torch.int32, device="cuda")
    pkg.token_logprobs(x, tokens, lp)
    pkg.token_logprobs(x, None, None, ent)
    pkg.token_logprobs(x, None, None, None, ids)
    pkg.token_logprobs(x, None, None, None, None, tops)
    for got, w in ((lp, want[0]), (ent, want[1]), (tops, want[3])):
        assert torch.allclose(got.double().cpu(), w, atol=1e-4)
    assert torch.equal(ids.cpu().long(), want[2])
    pkg.token_logprobs(x[:0], tokens[:0], lp[:0])          # no rows: nothing to do


# ---------------------------------------------------------------------------------------------- scoring with a model

@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_score_of_a_language_model(pkg, dtype):
    """What score says is what step's logits say: portions of several blocks, single tokens (launched, captured, replayed), any places."""
    import numpy as np
    from lm_models import attention, config, delta, tokens
    c = config([delta(), attention()])
    with pkg.LanguageModel(config=c, dtype=dtype, seed=3, max_tokens=400, max_seqs=2, block_rows=100) as lm:
        t = np.asarray(tokens(c, 260, 5))
        a, b = lm.open(), lm.open()
        cuts = [(0, 230), (230, 231), (231, 232), (232, 233), (233, 236), (236, 260)]
        for i, j in cuts:
            part, top = t[i:j], min(7, c["vocab"]) if i % 2 else 0
            want = list(range(j - i)) if j - i < 200 else [0, 5, 99, 100, 163, 164, 165, 229]
            targets = [int(t[min(i + w + 1, 259)]) for w in want]
            x = lm.step(a, part, want=want)
            lp, ent, ids, tops = lm.score(b, part, want=want, targets=targets, top=top)
            w_lp, w_ent, w_ids, w_tops = plain.logprobs(torch.from_numpy(x), torch.tensor(targets), top)
            assert np.allclose(lp, w_lp.numpy(), atol=1e-4) and np.allclose(ent, w_ent.numpy(), atol=1e-3)
            assert np.array_equal(ids, w_ids.numpy()) and np.allclose(tops, w_tops.numpy(), atol=1e-4)
            assert lm.length(a) == lm.length(b) == j
        lm.release(b)
        b = lm.open()
        lp, _, _, _ = lm.score(b, t[:150])
        assert lp.shape == (149,)
        for args in (dict(want=[3, 2], targets=[0, 0]), dict(want=[0], targets=[c["vocab"]]), dict(want=[0], targets=[-1]), dict(want=[0], targets=[0], top=33)):
            with pytest.raises(RuntimeError):
                lm.score(b, t[:5], **args)
        for args in (dict(want=[0]), dict(want=[0, 1], targets=[0]), dict(want=[], targets=[])):
            with pytest.raises(ValueError):
                lm.score(b, t[:5], **args)
        assert lm.length(b) == 150
