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
