"""Operators of a server of language models, as cases of stated sizes: a key/value cache held in 4 bits (append, attention),
eviction from it by accumulated attention weight, log probabilities of tokens out of logits.

    listed()            the cases
    draw(rng)           another case of the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass: the framework's calls where `own` is true, elementary torch operations where it is not
    work(case)          the bytes and operations that a pass cannot do without
    exact(case, seed)   what run returns, in 64 bits

The cache's format: a row of a head in blocks of 32 values; a block has a scale 2^e, e = floor(log2(largest magnitude)) - 2 (not
below -126), and its values are rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times that, ties to the even code."""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAME = "voxtral_tts_c_b200"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def package():
    if NAME not in sys.modules:
        folder = os.path.join(ROOT, "voxtral-tts.c_b200")
        spec = importlib.util.spec_from_file_location(NAME, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        sys.modules[NAME] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[NAME])
    return sys.modules[NAME]


# ---------------------------------------------------------------------------------------------- the cases

def _attend(name, seqs, rows, heads, kv_heads, dim, length, dtype, mass=False):
    return {"name": name, "op": "attend", "seqs": seqs, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "length": length, "dtype": dtype,
            "mass": mass}


def _append(name, seqs, rows, kv_heads, dim, length, dtype):
    return {"name": name, "op": "append", "seqs": seqs, "rows": rows, "kv_heads": kv_heads, "dim": dim, "length": length, "dtype": dtype}


def _evict(name, seqs, kv_heads, dim, length, keep, recent, first):
    return {"name": name, "op": "evict", "seqs": seqs, "kv_heads": kv_heads, "dim": dim, "length": length, "keep": keep, "recent": recent, "first": first}


def _logprobs(name, rows, vocab, top, dtype):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype}


def listed():
    return [
        # one token of the speech decoder (its heads) in the middle of an utterance, fp32 as its rows are: latency
        _attend("attend_step", 1, 1, 32, 8, 128, 301, "float32"),
        # one token of eight sequences of a language model at unequal lengths, whose weights an eviction will read
        _attend("attend_batch", 8, 1, 32, 8, 128, 4608, "bfloat16", True),
        # one token of four sequences with very long contexts
        _attend("attend_long", 4, 1, 32, 8, 128, 131072, "bfloat16"),
        # five drafted tokens to be checked, of a model with small heads and a large group
        _attend("attend_draft", 3, 5, 12, 2, 64, 2050, "float16", True),
        # a portion of a prompt that continues a cached one
        _attend("attend_prompt", 1, 1203, 32, 8, 128, 4208, "float32"),
        # the token's keys and values into the caches of eight sequences
        _append("append_step", 8, 1, 8, 128, 4608, "float32"),
        # a prompt's keys and values
        _append("append_prompt", 2, 4097, 8, 128, 8192, "bfloat16"),
        # one sequence back to its budget
        _evict("evict_one", 1, 8, 128, 1601, 1024, 256, 4),
        # sixteen long sequences to a quarter of their length
        _evict("evict_many", 16, 8, 128, 32768, 8192, 1024, 4),
        # one row of logits of the speech model's vocabulary, sampled by the caller
        _logprobs("logprobs_token", 1, 131072, 5, "float32"),
        # a lock-step batch with alternatives
        _logprobs("logprobs_batch", 64, 131072, 20, "bfloat16"),
        # a document scored at once, odd vocabulary
        _logprobs("logprobs_document", 1024, 100003, 1, "float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "evict", "logprobs"])
    dtype = rng.choice(list(TYPES))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 96, 128, 128, 192, 256])
    if op == "attend":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
        rows = rng.choice([1, 1, 1, rng.randint(2, 16), _log_int(rng, 17, 1024)])
        length = max(rows, _log_int(rng, 1, 65536 if rows <= 16 else 4096))
        # no more keys than the longest listed case has, no more products than the listed prompt
        length = max(rows, min(length, 1203 * 32 * 4208 * 128 // (rows * heads * dim)))
        most = min(4 * 8 * 131072 * 128 // (kv_heads * length * dim), 1203 * 32 * 4208 * 128 // (rows * heads * length * dim))
        return {"op": op, "seqs": rng.randint(1, max(1, min(16, most))), "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "length": length,
                "dtype": dtype, "mass": rng.random() < 0.4}
    if op == "append":
        rows = _log_int(rng, 1, 4097)
        return {"op": op, "seqs": rng.randint(1, 16 if rows < 512 else 2), "rows": rows, "kv_heads": kv_heads, "dim": dim,
                "length": rows + rng.randint(0, 1000), "dtype": dtype}
    if op == "evict":
        length = _log_int(rng, 16, 32768)
        keep = rng.randint(max(2, length // 8), length)
        return {"op": op, "seqs": rng.randint(1, 8), "kv_heads": kv_heads, "dim": dim, "length": length, "keep": keep, "recent": rng.randint(0, keep // 2),
                "first": rng.randint(0, min(4, keep // 2))}
    vocab = _log_int(rng, 100, 262144)
    return {"op": op, "rows": _log_int(rng, 1, max(1, min(1024, 100000000 // vocab))), "vocab": vocab, "top": min(vocab, rng.choice([0, 1, 5, 20, 32])),
            "dtype": dtype}


def _lengths(case):
    """Tokens in the cache of each sequence: the first has the case's length, the others between half of it and all."""
    n, least = case["length"], case.get("rows", 1)
    return [max(least, n - (n // 2) * i // max(1, case["seqs"] - 1)) for i in range(case["seqs"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _made(case, seed):
    """The inputs that a seed stands for."""
    g = _generator(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "logprobs":
        # peaked rows, as a model's are: a few tokens far above the others
        x = normal(case["rows"], case["vocab"]) * 2.0
        at = torch.randint(case["vocab"], (case["rows"], 16), generator=g, device="cuda")
        x.scatter_add_(1, at, normal(case["rows"], 16).abs() * 6.0)
        tokens = torch.where(torch.rand(case["rows"], generator=g, device="cuda") < 0.5, at[:, 0], torch.randint(case["vocab"], (case["rows"],), generator=g, device="cuda"))
        return {"logits": x.to(TYPES[case["dtype"]]), "tokens": tokens.to(torch.int32)}
    b, h, d, n = case["seqs"], case["kv_heads"], case["dim"], case["length"]
    lengths = _lengths(case)
    made = {"lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "n": lengths}
    dtype = TYPES[case["dtype"]] if "dtype" in case else torch.bfloat16
    # keys have a few channels of large magnitude, values none
    gain = 1.0 + 3.0 * (torch.rand(h, d, generator=g, device="cuda") < 0.05)
    rows = case["rows"] if case["op"] == "append" else n
    made["k"] = (normal(b, rows, h, d) * gain).to(dtype)
    made["v"] = normal(b, rows, h, d).to(dtype)
    if case["op"] == "attend":
        made["q"] = normal(b, case["rows"], case["heads"], d).to(dtype)
        made["mass"] = torch.rand(b, h, n, generator=g, device="cuda") if case["mass"] else None
    if case["op"] == "evict":
        # weights as attention leaves them: most of them small, over several magnitudes
        made["mass"] = torch.exp(normal(b, h, n) * 2.0 - 4.0)
    return made


# ---------------------------------------------------------------------------------------------- the plain form

def _levels(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=device)


def _quantise(x):
    """Rows [..., D] as codes [..., D / 2] (two a byte, the first value in the low half) and scale bytes [..., D / 32]."""
    x = x.float().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -126).clamp(min=-126)
    r = torch.ldexp(x, -e)
    a = r.abs()
    # codes 0 to 4 are steps of a half, 4 to 6 of one, 6 and 7 of two
    c = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4)).clamp(max=7)
    c = (c + torch.where(torch.signbit(r), 8.0, 0.0)).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), (e + 127).squeeze(-1).to(torch.uint8)


def _values(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = _levels(c.device)[c.int()].unflatten(-1, (-1, 32))
    return (x * torch.exp2(scales.float() - 127.0)[..., None]).flatten(-2)


def _plain_attend(s):
    case, out = s["case"], {}
    t, g, n = case["rows"], case["heads"] // case["kv_heads"], case["length"]
    k, v = _values(s["k_codes"], s["k_scales"]), _values(s["v_codes"], s["v_scales"])       # [B, H, n, D]
    b, h, _, d = k.shape
    q = s["q"].float().unflatten(2, (h, g)).permute(0, 2, 3, 1, 4).reshape(b, h, g * t, d)
    x = torch.matmul(q, k.transpose(-1, -2)) * case["dim"] ** -0.5
    row = torch.arange(t, device=x.device).repeat(g)
    sees = torch.arange(n, device=x.device)[None, None] <= (s["lengths"][:, None, None] - t + row[None, :, None])
    x.masked_fill_(~sees[:, None], float("-inf"))
    most = x.amax(-1, keepdim=True)
    x = torch.exp(x - most)
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v) / total
    out["lse"] = (most + torch.log(total)).unflatten(2, (g, t)).permute(0, 3, 1, 2, 4).reshape(b, t, h * g)
    out["out"] = o.unflatten(2, (g, t)).permute(0, 3, 1, 2, 4).reshape(b, t, h * g, d).to(s["q"].dtype)
    if s["mass"] is not None:
        at = torch.arange(n, device=x.device)[None, None]
        length = s["lengths"][:, None, None]
        m = torch.where(at < length - t, s["mass"], 0.0) + (x / total).sum(2)
        out["mass"] = torch.where(at < length, m, 0.0)
    return out


def _plain_append(s):
    b, t = s["k"].shape[:2]
    out, at = {}, s["at"]
    for name in ("k", "v"):
        c, e = _quantise(s[name])
        s[name + "_codes"][s["seq"], :, at] = c
        s[name + "_scales"][s["seq"], :, at] = e
        out[name] = _values(s[name + "_codes"][s["seq"], :, at], s[name + "_scales"][s["seq"], :, at])
    return out


def _plain_evict(s):
    case = s["case"]
    n, keep, first, recent = s["lengths"].long()[:, None, None], case["keep"], case["first"], case["recent"]
    b, h, most = s["mass"].shape
    at = torch.arange(most, device="cuda")[None, None]
    m = torch.where((at < first) | (at >= n - recent), float("inf"), s["mass"])
    m = torch.where(at < n, m, float("-inf"))
    order = torch.sort(m, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = torch.minimum(n, torch.tensor(keep, device="cuda"))
    place = torch.arange(keep, device="cuda")[None, None]
    kept = torch.sort(torch.where(place < count, order, most), dim=-1).values
    there = place < count
    i = torch.where(there, kept, 0)
    out = {"kept": torch.where(there, kept, -1).to(torch.int32), "lengths": count[:, 0, 0].to(torch.int32), "mass": torch.where(there, s["mass"].gather(2, i), 0.0)}
    for name in ("k", "v"):
        c, e = s[name + "_codes"], s[name + "_scales"]
        x = _values(c.gather(2, i[..., None].expand(-1, -1, -1, c.shape[-1])), e.gather(2, i[..., None].expand(-1, -1, -1, e.shape[-1])))
        out[name] = torch.where(there[..., None], x, 0.0).transpose(1, 2).to(torch.bfloat16)
    return out


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    out = {"logprobs": (x.gather(1, s["tokens"].long()[:, None]) - m - lse)[:, 0], "entropy": (lse - (e * (x - m)).sum(-1, keepdim=True) / total)[:, 0]}
    if top:
        v, i = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_ids"], out["top_logprobs"] = i[:, :top].to(torch.int32), v[:, :top] - m - lse
    return out


# ---------------------------------------------------------------------------------------------- what a program has in hand

def _filled(case, made, capacity):
    """A cache of the framework that holds the keys and values made."""
    cache = package().KV4Cache(case["seqs"], case["kv_heads"], case["dim"], capacity)
    full = torch.full((case["seqs"],), case["length"], dtype=torch.int32, device="cuda")
    cache.append(made["k"], made["v"], full)
    torch.cuda.synchronize()
    return cache


def prepare(case, seed):
    made, op = _made(case, seed), case["op"]
    s = {"case": case}
    if op == "logprobs":
        rows, top = case["rows"], case["top"]
        s.update(made)
        if own:
            s["logprobs"], s["entropy"] = (torch.empty(rows, device="cuda") for _ in range(2))
            if top:
                s["top_ids"] = torch.empty(rows, top, dtype=torch.int32, device="cuda")
                s["top_logprobs"] = torch.empty(rows, top, device="cuda")
            s["call"] = package().token_logprobs_call(made["logits"], made["tokens"], s["logprobs"], s["entropy"], s.get("top_ids"), s.get("top_logprobs"))
        return s
    b, h, d, n = case["seqs"], case["kv_heads"], case["dim"], case["length"]
    s["lengths"] = made["lengths"]
    if op == "append":
        s.update(k=made["k"], v=made["v"])
        if own:
            s["cache"] = package().KV4Cache(b, h, d, n)
            s["out"] = {"k": torch.empty(b, case["rows"], h, d, device="cuda"), "v": torch.empty(b, case["rows"], h, d, device="cuda")}
            s["call"] = s["cache"].append_call(made["k"], made["v"], made["lengths"])
            s["read"] = s["cache"].read_call(s["out"]["k"], s["out"]["v"], made["lengths"])
        else:
            for name in ("k", "v"):
                s[name + "_codes"] = torch.zeros(b, h, n, d // 2, dtype=torch.uint8, device="cuda")
                s[name + "_scales"] = torch.zeros(b, h, n, d // 32, dtype=torch.uint8, device="cuda")
            s["seq"] = torch.arange(b, device="cuda")[:, None]
            s["at"] = made["lengths"].long()[:, None] - case["rows"] + torch.arange(case["rows"], device="cuda")[None]
        return s
    s["mass"] = made["mass"]
    if op == "attend":
        s["q"] = made["q"]
    if not own:
        for name in ("k", "v"):
            c, e = _quantise(made[name])
            s[name + "_codes"], s[name + "_scales"] = c.transpose(1, 2).contiguous(), e.transpose(1, 2).contiguous()
        return s
    s["cache"] = _filled(case, made, n)
    if op == "attend":
        s["out"] = {"out": torch.empty_like(made["q"]), "lse": torch.empty(b, case["rows"], case["heads"], device="cuda")}
        if case["mass"]:
            s["out"]["mass"] = torch.zeros_like(made["mass"])
        s["call"] = s["cache"].attention_call(made["q"], s["out"]["out"], made["lengths"], scale=d ** -0.5, lse=s["out"]["lse"],
                                               mass_in=made["mass"], mass_out=s["out"].get("mass"))
    else:
        keep = case["keep"]
        s["into"] = package().KV4Cache(b, h, d, keep)
        s["out"] = {"kept": torch.full((b, h, keep), -1, dtype=torch.int32, device="cuda"), "lengths": torch.empty(b, dtype=torch.int32, device="cuda"),
                    "mass": torch.zeros(b, h, keep, device="cuda"), "k": torch.zeros(b, keep, h, d, dtype=torch.bfloat16, device="cuda"),
                    "v": torch.zeros(b, keep, h, d, dtype=torch.bfloat16, device="cuda")}
        s["call"] = s["cache"].evict_call(s["into"], made["lengths"], s["out"]["lengths"], made["mass"], s["out"]["mass"], keep=keep, recent=case["recent"],
                                          first=case["first"], kept=s["out"]["kept"])
        s["read"] = s["into"].read_call(s["out"]["k"], s["out"]["v"], s["out"]["lengths"], rows=s["out"]["lengths"])
    return s


# ---------------------------------------------------------------------------------------------- one pass

PLAIN = {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict, "logprobs": _plain_logprobs}


def run(state):
    if not own:
        return PLAIN[state["case"]["op"]](state)
    state["call"]()
    if "read" in state:
        state["read"]()
    if state["case"]["op"] == "logprobs":
        return {k: state[k] for k in ("logprobs", "entropy", "top_ids", "top_logprobs") if k in state}
    return state["out"]


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    size = TYPES[case["dtype"]].itemsize if "dtype" in case else 2
    if op == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": rows * vocab * size + rows * (12 + 8 * top), "flops": 5 * rows * vocab}
    b, h, d = case["seqs"], case["kv_heads"], case["dim"]
    row = h * (d + d // 16)                       # a token's codes and scales, keys and values
    lengths = _lengths(case)
    if op == "append":
        t = b * case["rows"]
        return {"bytes": 2 * t * h * d * size + 2 * t * row + 2 * t * h * d * 4, "flops": 8 * t * h * d}
    if op == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": sum(lengths) * h * 4 + kept * (2 * row + 8 * h + 2 * h * d * 2), "flops": sum(lengths) * h}
    t, heads = case["rows"], case["heads"]
    pairs = sum(t * n - t * (t - 1) // 2 for n in lengths)
    moved = sum(lengths) * row + 2 * b * t * heads * d * size + b * t * heads * 4
    if case["mass"]:
        moved += sum(lengths) * h * 8
    return {"bytes": moved, "flops": 4 * pairs * heads * d}


# ---------------------------------------------------------------------------------------------- 64 bits

def _exact_rounded(x):
    """Values of rows [..., D] as the cache stands for them, by comparison with the borders between neighbouring levels."""
    x = x.double().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(most.clamp(min=2.0 ** -130)))
    e = torch.where(torch.exp2(e) > most, e - 1, torch.where(torch.exp2(e + 1) <= most, e + 1, e))
    unit = torch.exp2((e - 2).clamp(min=-126))
    a, y = x.abs() / unit, torch.zeros_like(x)
    # a border belongs to the level with the even code: above it (">=") where that is the upper one
    for border, level, upper in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True), (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
        y = torch.where(a >= border if upper else a > border, level, y)
    return (torch.copysign(y, x) * unit).flatten(-2)


def exact(case, seed):
    made, op = _made(case, seed), case["op"]
    if op == "logprobs":
        top, out = case["top"], {"logprobs": [], "entropy": [], "top_ids": [], "top_logprobs": []}
        for r in range(0, case["rows"], 64):
            x = made["logits"][r:r + 64].double()
            lp = torch.log_softmax(x, -1)
            out["logprobs"].append(lp.gather(1, made["tokens"][r:r + 64].long()[:, None])[:, 0])
            out["entropy"].append(-(lp.exp() * lp).sum(-1))
            if top:
                i = torch.sort(-x, dim=-1, stable=True).indices[:, :top]
                out["top_ids"].append(i.to(torch.int32))
                out["top_logprobs"].append(lp.gather(1, i))
        return {k: torch.cat(v) for k, v in out.items() if v}
    if op == "append":
        return {"k": _exact_rounded(made["k"]), "v": _exact_rounded(made["v"])}
    if op == "evict":
        b, h, keep = case["seqs"], case["kv_heads"], case["keep"]
        out = {"kept": torch.full((b, h, keep), -1, dtype=torch.int32, device="cuda"), "mass": torch.zeros(b, h, keep, dtype=torch.float64, device="cuda")}
        for name in ("k", "v"):
            out[name] = torch.zeros(b, keep, h, case["dim"], dtype=torch.float64, device="cuda")
        for i, n in enumerate(made["n"]):
            count = min(n, keep)
            for j in range(h):
                m = made["mass"][i, j, :n].double()
                if n <= keep:
                    kept = torch.arange(n, device="cuda")
                else:
                    first, recent = case["first"], case["recent"]
                    middle = torch.sort(-m[first:n - recent], stable=True).indices[:keep - first - recent] + first
                    kept = torch.cat((torch.arange(first, device="cuda"), middle.sort().values, torch.arange(n - recent, n, device="cuda")))
                out["kept"][i, j, :count] = kept.to(torch.int32)
                out["mass"][i, j, :count] = m[kept]
                for name in ("k", "v"):
                    out[name][i, :count, j] = _exact_rounded(made[name][i, kept, j])
        out["lengths"] = torch.tensor([min(n, keep) for n in made["n"]], dtype=torch.int32, device="cuda")
        return out
    t, heads, h, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    g = heads // h
    out = {"out": torch.zeros(case["seqs"], t, heads, d, dtype=torch.float64, device="cuda"), "lse": torch.zeros(case["seqs"], t, heads, dtype=torch.float64, device="cuda")}
    if case["mass"]:
        out["mass"] = torch.zeros(case["seqs"], h, case["length"], dtype=torch.float64, device="cuda")
    for i, n in enumerate(made["n"]):
        for j in range(h):
            k, v = _exact_rounded(made["k"][i, :n, j]), _exact_rounded(made["v"][i, :n, j])
            hidden = torch.ones(t, n, dtype=torch.bool, device="cuda").triu(n - t + 1)
            if case["mass"]:
                out["mass"][i, j, :n - t] = made["mass"][i, j, :n - t].double()
            for u in range(j * g, j * g + g):
                x = (made["q"][i, :, u].double() @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                out["lse"][i, :, u] = torch.logsumexp(x, -1)
                p = torch.softmax(x, -1)
                out["out"][i, :, u] = p @ v
                if case["mass"]:
                    out["mass"][i, j, :n] += p.sum(0)
    return out
