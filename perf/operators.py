"""The attention block of a decoder that is being served, operator by operator, as timed cases.

Five operators, in the order in which a layer calls them:

* ``quantize``:  ``eager.quantize_rows`` - rows of activations to 8-bit integers with a scale for each row;
* ``int8``:      ``eager.gemm_rcr_int8`` - the product of such rows with an 8-bit weight that has a scale for each channel;
* ``rotary``:    ``eager.rotary_embedding`` - positions rotated into the heads (and back: its gradient);
* ``append``:    ``eager.paged_kv_append`` - new keys and values into a paged cache, keys and queries rotated on the way;
* ``attention``: ``eager.prefix_attention`` - queries against a prefix that the whole batch shares and each sequence's own pages.

Where ``own`` is false, ``run`` computes them from elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # the activations of 64 sequences that decode one token each, ahead of a projection
        {"name": "quantize_decode", "path": "quantize", "dtype": "float16", "rows": 64, "columns": 4096},
        # the same over 16384 tokens of prompts
        {"name": "quantize_prompt", "path": "quantize", "dtype": "bfloat16", "rows": 16384, "columns": 8192},
        # one token through a projection: all of it is reading the weight
        {"name": "int8_one_row", "path": "int8", "dtype": "float16", "M": 1, "N": 4096, "K": 4096, "bias": True},
        # a short prompt through a layer whose sizes divide by nothing (rows of the operands at any byte)
        {"name": "int8_ragged", "path": "int8", "dtype": "bfloat16", "M": 777, "N": 2731, "K": 1101, "bias": True},
        # the largest dense product of the GEMM benchmark, in 8 bits
        {"name": "int8_square", "path": "int8", "dtype": "bfloat16", "M": 8192, "N": 8192, "K": 8192, "bias": False},
        # the queries of eight sequences that decode, far into a long context
        {"name": "rotary_decode", "path": "rotary", "dtype": "float16", "tokens": 8, "heads": 16, "head_dim": 128, "rotated": 128,
         "interleaved": False, "furthest": 1 << 20, "inverse": False},
        # a prompt: neighbouring dims rotated, in a part of each head, the rest handed through
        {"name": "rotary_prompt", "path": "rotary", "dtype": "bfloat16", "tokens": 16384, "heads": 32, "head_dim": 128, "rotated": 64,
         "interleaved": True, "furthest": 1 << 15, "inverse": False},
        # one token each of 64 sequences, grouped heads, into pages of 16
        {"name": "append_decode", "path": "append", "dtype": "float16", "batch": 64, "most": 1, "least": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rotated": 128, "interleaved": False, "page": 16, "past": 4096, "heads_first": False},
        # eight prompts of 517 to 2048 tokens, pages that lie head by head
        {"name": "append_prompts", "path": "append", "dtype": "bfloat16", "batch": 8, "most": 2048, "least": 517, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rotated": 128, "interleaved": False, "page": 64, "past": 64, "heads_first": True},
        # one sequence that decodes behind a short prompt
        {"name": "attention_one_token", "path": "attention", "dtype": "float16", "batch": 1, "most": 1, "least": 1, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "page": 16, "prefix": 384, "past": 61, "past_least": 61, "heads_first": False},
        # 64 sequences that decode, 32 to 1000 tokens each behind a prefix of 8192 that they share
        {"name": "attention_decode", "path": "attention", "dtype": "bfloat16", "batch": 64, "most": 1, "least": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "prefix": 8192, "past": 1000, "past_least": 32, "heads_first": False},
        # eight ragged pieces of prompts of 5 to 517 tokens behind a prefix that ends inside a page, narrow heads
        {"name": "attention_prompts", "path": "attention", "dtype": "float16", "batch": 8, "most": 517, "least": 5, "heads": 16,
         "kv_heads": 4, "head_dim": 80, "page": 64, "prefix": 2041, "past": 1333, "past_least": 0, "heads_first": True},
    ]


# ---- drawn cases -----------------------------------------------------------------------------------------------

def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice((1, 2, 4, 8))
    return kv * rng.choice((1, 1, 2, 4, 7, 8)), kv


def _draw_quantize(rng):
    return {"path": "quantize", "dtype": rng.choice(sorted(DTYPES)), "rows": _log(rng, 1, 16384), "columns": _log(rng, 64, 8192)}


def _draw_int8(rng):
    some = (lambda: _log(rng, 64, 8192)) if rng.random() < 0.3 else (lambda: max(16, _log(rng, 64, 8192) // 16 * 16))
    return {"path": "int8", "dtype": rng.choice(sorted(DTYPES)), "M": _log(rng, 1, 8192), "N": some(), "K": some(),
            "bias": rng.random() < 0.5}


def _draw_rotary(rng):
    head_dim = rng.choice((64, 80, 96, 128, 256))
    return {"path": "rotary", "dtype": rng.choice(sorted(DTYPES)), "tokens": _log(rng, 1, 16384), "heads": rng.choice((1, 4, 12, 16, 32)),
            "head_dim": head_dim, "rotated": rng.choice((head_dim, head_dim // 2)), "interleaved": rng.random() < 0.5,
            "furthest": _log(rng, 1 << 11, 1 << 20), "inverse": rng.random() < 0.4}


def _draw_append(rng):
    heads, kv_heads = _heads(rng)
    head_dim, most = rng.choice((64, 80, 128)), 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    return {"path": "append", "dtype": rng.choice(sorted(DTYPES)), "batch": _log(rng, 1, 64), "most": most, "least": rng.randint(1, most),
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotated": rng.choice((0, head_dim // 2, head_dim)),
            "interleaved": rng.random() < 0.5, "page": rng.choice((16, 32, 64, 256)), "past": _log(rng, 1, 4096),
            "heads_first": rng.random() < 0.5}


def _draw_attention(rng):
    heads, kv_heads = _heads(rng)
    most, past = 1 if rng.random() < 0.6 else _log(rng, 2, 517), _log(rng, 1, 4096)
    return {"path": "attention", "dtype": rng.choice(sorted(DTYPES)), "batch": _log(rng, 1, 64), "most": most,
            "least": rng.randint(1, most), "heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice((64, 80, 96, 128)),
            "page": rng.choice((16, 32, 64, 256)), "prefix": rng.choice((0, _log(rng, 1, 8192), _log(rng, 1, 8192))), "past": past,
            "past_least": rng.randint(0, past), "heads_first": rng.random() < 0.5}


def draw(rng):
    kinds = {"quantize": _draw_quantize, "int8": _draw_int8, "rotary": _draw_rotary, "append": _draw_append, "attention": _draw_attention}
    path = rng.choice(sorted(kinds))
    most = [work(c) for c in listed() if c["path"] == path]
    while True:
        case = kinds[path](rng)
        w = work(case)
        # (a plain form of attention holds all scores of the padded batch)
        if (w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most)
                and (path != "attention" or case["batch"] * case["most"] * case["heads"] * (case["prefix"] + case["past"] + case["most"]) < 1 << 28)):
            return case


# ---- work ------------------------------------------------------------------------------------------------------

def _spread(least, most, n):
    """n numbers from `most` down to `least`, evenly."""
    return [most - (most - least) * i // max(1, n - 1) for i in range(n)]


def work(case):
    if case["path"] == "quantize":
        n = case["rows"] * case["columns"]
        return {"bytes": 3 * n + 4 * case["rows"], "flops": 3 * n}
    if case["path"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 2 * M * N + 4 * (M + N) + 2 * N * case["bias"], "flops": 2 * M * N * K}
    if case["path"] == "rotary":
        n = case["tokens"] * case["heads"]
        return {"bytes": 4 * n * case["head_dim"] + 8 * case["tokens"] + 2 * case["rotated"], "flops": 3 * n * case["rotated"]}
    new = _spread(case["least"], case["most"], case["batch"])
    if case["path"] == "append":
        n = sum(new)
        return {"bytes": 4 * n * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"] + 8 * case["batch"],
                "flops": 3 * n * (case["heads"] + case["kv_heads"]) * case["rotated"]}
    past, D = _spread(case["past_least"], case["past"], case["batch"]), case["head_dim"]
    keys = case["prefix"] + sum(p + n for p, n in zip(past, new))
    pairs = sum(n * (case["prefix"] + p) + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": 4 * D * (case["kv_heads"] * keys + case["heads"] * sum(new)), "flops": 4 * D * case["heads"] * pairs}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _frequencies(rotated):
    return (10000.0 ** (torch.arange(0, rotated, 2, dtype=torch.float64, device="cuda") / -max(1, rotated))).float()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(dtype)

    def whole(*shape):
        return torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8)

    def positive(n):
        return torch.rand(n, device="cuda", generator=g).add_(0.5).mul_(0.01)

    s = {"path": case["path"]}
    if case["path"] == "quantize":
        # rows of different sizes, a few columns larger than the rest
        s["x"] = normal(case["rows"], case["columns"])
        s["x"] *= torch.rand(case["rows"], 1, device="cuda", generator=g).add_(0.1).to(dtype)
        s["x"][:, ::61] *= 8
        return s
    if case["path"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        s.update(a=whole(M, K), b=whole(N, K), a_scale=positive(M), b_scale=positive(N), bias=normal(N) if case["bias"] else None,
                 dtype=dtype)
        return s
    if case["path"] == "rotary":
        s.update(x=normal(case["tokens"], case["heads"], case["head_dim"]), freqs=_frequencies(case["rotated"]),
                 positions=torch.randint(0, case["furthest"], (case["tokens"],), device="cuda", generator=g),
                 interleaved=case["interleaved"], inverse=case["inverse"], scale=1.0)
        return s
    B, H, C, D, page = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim", "page"))
    new = _spread(case["least"], case["most"], B)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    past = [case["past"]] * B if case["path"] == "append" else _spread(case["past_least"], case["past"], B)
    # pages dealt out of order; the first of them are the prefix's
    prefix = case.get("prefix", 0)
    held = [-(-(p + n) // page) for p, n in zip(past, new)]
    prefix_pages = -(-prefix // page)
    pages = prefix_pages + sum(held) + 2
    order = torch.randperm(pages, device="cuda", generator=g, dtype=torch.int32)
    table = torch.full((B, max(held)), -1, dtype=torch.int32, device="cuda")
    taken = torch.arange(max(held), device="cuda")[None, :] < torch.tensor(held, device="cuda")[:, None]
    table[taken] = order[prefix_pages:prefix_pages + sum(held)]
    s.update(table=table, lengths=_ints(past), offsets=_ints(offsets) if case["most"] > 1 else None, most=case["most"], new=_ints(new))
    shape = (pages, C, page, D) if case["heads_first"] else (pages, page, C, D)
    k_cache, v_cache = normal(*shape), normal(*shape)
    s["k_cache"], s["v_cache"] = (k_cache.transpose(1, 2), v_cache.transpose(1, 2)) if case["heads_first"] else (k_cache, v_cache)
    if case["path"] == "append":
        # queries, keys and values as one projection leaves them
        qkv = normal(offsets[-1], H + 2 * C, D)
        s.update(q=qkv[:, :H], k=qkv[:, H:H + C], v=qkv[:, H + C:], interleaved=case["interleaved"],
                 freqs=_frequencies(case["rotated"]) if case["rotated"] else None)
        return s
    s.update(q=normal(offsets[-1], H, D), prefix=prefix, prefix_table=order[:prefix_pages] if prefix else None)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------

def _rotate(x, positions, freqs, interleaved, inverse=False, scale=1.0):
    """x [tokens, heads, dim] in 32 bits; the angles of far positions take 64."""
    n = freqs.numel()
    angle = positions.double()[:, None] * freqs.double()
    cos, sin = (angle.cos() * scale).float()[:, None], (angle.sin() * scale).float()[:, None]
    sin = -sin if inverse else sin
    one, two = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    a, b = one * cos - two * sin, two * cos + one * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _places(s):
    """(sequence, place among its own tokens) of each row."""
    rows = torch.arange(s["q"].shape[0], device="cuda")
    if s["offsets"] is None:
        return rows, s["lengths"].long()
    seq = torch.searchsorted(s["offsets"], rows, right=True) - 1
    return seq, s["lengths"][seq] + rows - s["offsets"][seq]


def _plain_append(s):
    seq, place = _places(s)
    page = s["k_cache"].shape[1]
    at = s["table"][seq, place // page].long(), place % page
    q, k = s["q"], s["k"]
    if s["freqs"] is not None:
        q, k = (_rotate(x.float(), place, s["freqs"], s["interleaved"]).to(x.dtype) for x in (q, k))
    s["k_cache"][at] = k
    s["v_cache"][at] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_attention(s):
    q, C, D, page = s["q"], s["k_cache"].shape[2], s["q"].shape[2], s["k_cache"].shape[1]
    T, H = q.shape[:2]
    B, N, P, L = s["table"].shape[0], s["most"], s["prefix"], s["table"].shape[1] * page
    G = H // C
    # queries padded to the longest sequence's: [B, C, N * G, D]
    first = s["offsets"][:-1].long() if s["offsets"] is not None else torch.arange(B, device="cuda")
    step = torch.arange(N, device="cuda")
    rows = (first[:, None] + step).clamp(max=T - 1)
    x = q.float()[rows].view(B, N, C, G, D).permute(0, 2, 1, 3, 4).reshape(B, C, N * G, D) * D ** -0.5
    seen = s["lengths"].long()[:, None] + step + 1  # [B, N] own keys that a row sees
    there = torch.arange(L, device="cuda") < seen[:, -1:]  # ... and that any row of the sequence does
    pages = s["table"].clamp(min=0).long()
    k, v = (c[pages].reshape(B, L, C, D).float().permute(0, 2, 1, 3) for c in (s["k_cache"], s["v_cache"]))
    v = v.masked_fill(~there[:, None, :, None], 0.0)
    score = torch.matmul(x, k.transpose(2, 3).contiguous()).view(B, C, N, G, L)
    score = score.masked_fill((torch.arange(L, device="cuda") >= seen[:, :, None])[:, None, :, None], -math.inf).view(B, C, N * G, L)
    if P:
        flat = x.transpose(0, 1).reshape(C, B * N * G, D)
        pk, pv = (c[s["prefix_table"].long()].reshape(-1, C, D)[:P].float().transpose(0, 1) for c in (s["k_cache"], s["v_cache"]))
        shared = torch.matmul(flat, pk.transpose(1, 2).contiguous()).view(C, B, N * G, P).transpose(0, 1)
        score = torch.cat((shared, score), -1)
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    y = torch.matmul(p[..., P:], v.contiguous())
    if P:
        shared = p[..., :P].transpose(0, 1).reshape(C, B * N * G, P)
        y = y + torch.matmul(shared, pv.contiguous()).view(C, B, N * G, D).transpose(0, 1)
    y = y.view(B, C, N, G, D).permute(0, 2, 1, 3, 4).reshape(B, N, H, D).to(q.dtype)
    return y[:, 0] if N == 1 else y[step < s["new"][:, None]]


def run(s):
    if own:
        from aitemplate_amd import eager

        if s["path"] == "quantize":
            return eager.quantize_rows(s["x"])
        if s["path"] == "int8":
            return eager.gemm_rcr_int8(s["a"], s["b"], s["a_scale"], s["b_scale"], s["bias"], dtype=s["dtype"])
        if s["path"] == "rotary":
            return eager.rotary_embedding(s["x"], s["positions"], s["freqs"], interleaved=s["interleaved"], inverse=s["inverse"],
                                          scale=s["scale"])
        if s["path"] == "append":
            q = eager.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["offsets"], q=s["q"],
                                      freqs=s["freqs"], interleaved=s["interleaved"])
            return q, s["k_cache"], s["v_cache"]
        return eager.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["offsets"],
                                      prefix_table=s["prefix_table"], prefix_length=s["prefix"])
    if s["path"] == "quantize":
        # (in 64 bits: quotients next to the middle of two whole numbers)
        x = s["x"].double()
        most = x.abs().amax(1, keepdim=True)
        q = (x * 127.0 / most).nan_to_num(0.0).round().to(torch.int8)
        return q, (most[:, 0] / 127.0).float()
    if s["path"] == "int8":
        # (in 64 bits: sums of more than 2^24)
        y = torch.matmul(s["a"].double(), s["b"].double().t()).float() * (s["a_scale"][:, None] * s["b_scale"])
        return (y if s["bias"] is None else y + s["bias"].float()).to(s["dtype"])
    if s["path"] == "rotary":
        return _rotate(s["x"].float(), s["positions"], s["freqs"], s["interleaved"], s["inverse"], s["scale"]).to(s["x"].dtype)
    return _plain_append(s) if s["path"] == "append" else _plain_attention(s)


# ---- what the operators are, in 64 bits ------------------------------------------------------------------------

def _exact_turn(x, positions, freqs, interleaved, inverse=False):
    """As products of complex numbers."""
    x, n = x.double(), freqs.numel()
    pairs = x[..., :2 * n].unflatten(-1, (n, 2)) if interleaved else x[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2)
    angle = positions.double().unsqueeze(-1) * freqs.double() * (-1.0 if inverse else 1.0)
    turned = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)
    turned = torch.view_as_real(turned)
    y = x.clone()
    y[..., :2 * n] = (turned if interleaved else turned.transpose(-1, -2)).reshape(*x.shape[:-1], 2 * n)
    return y


def _of_sequences(s):
    """(sequence, first row, rows, own tokens before them)."""
    past, new = s["lengths"].tolist(), s["new"].tolist()
    return [(b, sum(new[:b]), n, past[b]) for b, n in enumerate(new)]


def exact(case, seed):
    s = prepare(case, seed)
    if s["path"] == "quantize":
        scale = s["x"].double().abs().max(1).values / 127.0
        return None, scale
    if s["path"] == "int8":
        y = (s["a"].double() * s["a_scale"].double()[:, None]) @ (s["b"].double() * s["b_scale"].double()[:, None]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if s["path"] == "rotary":
        return _exact_turn(s["x"], s["positions"], s["freqs"], s["interleaved"], s["inverse"])
    page = s["k_cache"].shape[1]
    if s["path"] == "append":
        q, k, v = s["q"].double(), s["k_cache"].double(), s["v_cache"].double()
        q = q.clone()
        for b, row, n, past in _of_sequences(s):
            place = torch.arange(past, past + n, device="cuda")
            at = s["table"][b, place // page].long(), place % page
            if s["freqs"] is None:
                k[at] = s["k"][row:row + n].double()
            else:
                k[at] = _exact_turn(s["k"][row:row + n], place, s["freqs"], s["interleaved"])
                q[row:row + n] = _exact_turn(s["q"][row:row + n], place, s["freqs"], s["interleaved"])
            v[at] = s["v"][row:row + n].double()
        return q, k, v
    (T, H, D), C = s["q"].shape, s["k_cache"].shape[2]
    y = torch.empty(T, H, D, dtype=torch.float64, device="cuda")
    for b, row, n, past in _of_sequences(s):
        pages = s["table"][b, :-(-(past + n) // page)].long()
        keys = []
        for cache in (s["k_cache"], s["v_cache"]):
            mine = cache[pages].reshape(-1, C, D)[:past + n].double()
            if s["prefix"]:
                mine = torch.cat((cache[s["prefix_table"].long()].reshape(-1, C, D)[:s["prefix"]].double(), mine))
            keys.append(mine.repeat_interleave(H // C, 1).transpose(0, 1).contiguous())
        score = s["q"][row:row + n].double().transpose(0, 1) @ keys[0].transpose(1, 2) / math.sqrt(D)
        hidden = torch.ones(n, s["prefix"] + past + n, dtype=torch.bool, device="cuda").triu(s["prefix"] + past + 1)
        y[row:row + n] = (torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ keys[1]).transpose(0, 1)
    return y
