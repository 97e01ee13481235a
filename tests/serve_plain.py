"""The operators of voxtral_b200_serve.h in 64 bits, one sequence, head and row at a time, and how far a right kernel may be from them."""
import math

import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def rounded(x):
    """Rows [..., D] as the 4-bit cache stands for them; blocks with a value that is not finite are NaN."""
    x = x.double().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    safe = torch.where(bad | (most == 0), 1.0, most)
    e = torch.floor(torch.log2(safe))
    e = torch.where(torch.exp2(e) > safe, e - 1, torch.where(torch.exp2(e + 1) <= safe, e + 1, e))
    unit = torch.exp2((e - 2).clamp(min=-126.0))
    unit = torch.where(most == 0, 2.0 ** -126, unit)
    a, y = x.abs() / unit, torch.zeros_like(x)
    for i in range(7):          # a tie goes to the level with the even number
        border = (LEVELS[i] + LEVELS[i + 1]) / 2
        y = torch.where((a >= border) if (i + 1) % 2 == 0 else (a > border), LEVELS[i + 1], y)
    return torch.where(bad, math.nan, torch.copysign(y, x) * unit).flatten(-2)


def attention(q, k, v, length, rows, scale, mass_in=None):
    """One sequence: q [rows, heads, D]; k, v [H, n >= length, D] of the cache. Returns out, lse, mass [H, length], and the largest sum of
    |scale q_d k_d| of a score, the largest |v|."""
    q, k, v = q.double(), k.double()[:, :length], v.double()[:, :length]
    t, heads, d = q.shape
    h = k.shape[0]
    g = heads // h
    out = torch.zeros(t, heads, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, heads), -math.inf, dtype=torch.float64, device=q.device)
    mass = torch.zeros(h, length, dtype=torch.float64, device=q.device)
    if mass_in is not None:
        old = max(0, length - rows)
        mass[:, :old] = mass_in.double()[:, :old]
    for i in range(rows):
        sees = length - rows + i + 1
        if sees <= 0:
            continue
        for u in range(heads):
            s = (k[u // g, :sees] @ q[i, u]) * scale
            lse[i, u] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[i, u] = p @ v[u // g, :sees]
            mass[u // g, :sees] += p
    return out, lse, mass


def attention_bounds(q, k, v, scale, dtype):
    """(of a score, of a result apart from its own rounding) in absolute terms, from the kernels' roundings:

    a score    queries as two FP16 terms (2^-22 of a value; exact for bf16 and fp16, whose tiny values lose at most 2^-24 * 2^-14 of
               the row's largest), sums of 32 products in a tensor core and a block at a time beyond that: 2 * blocks + 4
               roundings at 2^-23 of the sum of magnitudes; times a constant in fp32, an exponential's argument: 4 * 2^-24 of the score
    a weight   twice a score's error, an exponential of 2^-21, one FP16 term (2^-11) for bf16 results, two (2^-21) otherwise, and FP16's
               smallest step (2^-24 of weights from 2^7 up) for every token
    a result   weights' error and (tokens / 16 + 8) sums at 2^-23, of the largest |v|"""
    q, k, v = q.double(), k.double(), v.double()
    n, d = k.shape[-2], k.shape[-1]
    sums = abs(scale) * float(q.abs().amax() * k.abs().sum(-1).amax()) if n else 0.0
    score = sums * ((2 * d // 32 + 4) * 2.0 ** -23 + 2.0 ** -22 + 4 * 2.0 ** -24 + 2.0 ** -21)
    term = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -21
    weight = 2 * score + 2.0 ** -21 + term + n * 2.0 ** -31
    most = float(v.abs().amax()) if n else 0.0
    return score + 2.0 ** -20, most * (weight + (n / 16 + 8) * 2.0 ** -23)


def kept(mass, n, keep, recent, first):
    """Which of n tokens stay, in order: a list."""
    if n <= keep:
        return list(range(n))
    m = [(-math.inf if math.isnan(x) else x) for x in mass[:n].double().tolist()]
    middle = sorted(range(first, n - recent), key=lambda i: (-m[i], i))[:keep - first - recent]
    return sorted(list(range(first)) + middle + list(range(n - recent, n)))


def logprobs(x, tokens, top):
    """Rows [rows, vocab]: log probabilities of the tokens, entropies, the largest values' indices and log probabilities."""
    y = x.double()
    rows, vocab = y.shape
    lp, ent = torch.full((rows,), math.nan, dtype=torch.float64), torch.full((rows,), math.nan, dtype=torch.float64)
    ids, tops = torch.zeros(rows, top, dtype=torch.int64), torch.zeros(rows, top, dtype=torch.float64)
    for r in range(rows):
        row = y[r]
        wrong = bool(torch.isnan(row).any() or (row == math.inf).any())
        order = torch.where(torch.isnan(row), math.inf, row)
        # NaN above +inf: two keys, the stable sort by the second first
        i = torch.sort(-order, stable=True).indices
        i = i[torch.sort((~torch.isnan(row[i])).int(), stable=True).indices][:top]
        ids[r] = i.cpu()
        token = int(tokens[r])
        known = 0 <= token < vocab
        if wrong:
            tops[r] = math.nan
        elif bool((row == -math.inf).all()):
            lp[r], ent[r], tops[r] = (-math.inf if known else math.nan), 0.0, -math.inf
        else:
            l = torch.log_softmax(row, 0)
            lp[r] = l[token] if known else math.nan
            p = l.exp()
            ent[r] = -(torch.where(p > 0, p * l, 0.0)).sum()
            tops[r] = l[i].cpu()
    return lp, ent, ids, tops
