"""What a served decoder computes around its attention, operator by operator, as timed cases.

In the order in which a step calls them:

* ``lora``:     ``eager.gemm_rcr_lora`` - a projection that all requests share, with the low-rank adapter of each row's request;
* ``norm``:     ``eager.qk_norm_rotary`` - queries and keys normalized head by head and rotated to their positions;
* ``append``:   ``eager.paged_kv_append`` with norms - the same on the way into a paged cache;
* ``logprobs``: ``eager.token_logprobs`` - log probabilities and ranks of given tokens, entropies, the most probable alternatives.

Where ``own`` is false, ``run`` computes them from elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
HALVES = ("bfloat16", "float16")
EPS = 1e-6


def listed():
    return [
        # one request that decodes, with an adapter of its own, through a square projection
        {"name": "lora_one_token", "path": "lora", "dtype": "float16", "rows": 1, "N": 4096, "K": 4096, "rank": 16, "adapters": 4,
         "requests": 1, "plain": 0, "bias": False},
        # 64 requests that decode beside each other, 48 adapters among them, eight requests without one
        {"name": "lora_decode", "path": "lora", "dtype": "bfloat16", "rows": 64, "N": 6144, "K": 4096, "rank": 16, "adapters": 48,
         "requests": 64, "plain": 8, "bias": False},
        # short prompts through a layer whose sizes divide by nothing much
        {"name": "lora_ragged", "path": "lora", "dtype": "float16", "rows": 777, "N": 2730, "K": 1100, "rank": 12, "adapters": 5,
         "requests": 7, "plain": 1, "bias": True},
        # long prompts of nine requests, wide adapters
        {"name": "lora_prompts", "path": "lora", "dtype": "bfloat16", "rows": 8192, "N": 8192, "K": 4096, "rank": 64, "adapters": 6,
         "requests": 9, "plain": 2, "bias": True},
        # the heads of 64 sequences that decode
        {"name": "norm_decode", "path": "norm", "dtype": "bfloat16", "tokens": 64, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rotated": 128, "interleaved": False, "furthest": 1 << 17},
        # 16384 tokens of prompts, half of each head rotated
        {"name": "norm_prompt", "path": "norm", "dtype": "float16", "tokens": 16384, "heads": 16, "kv_heads": 4, "head_dim": 256,
         "rotated": 128, "interleaved": True, "furthest": 1 << 15},
        # one token each of 48 sequences into pages of 16
        {"name": "append_decode", "path": "append", "dtype": "float16", "batch": 48, "most": 1, "least": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rotated": 128, "interleaved": False, "page": 16, "past": 4096, "heads_first": False},
        # eight prompts of 333 to 2048 tokens, pages that lie head by head
        {"name": "append_prompts", "path": "append", "dtype": "bfloat16", "batch": 8, "most": 2048, "least": 333, "heads": 32,
         "kv_heads": 4, "head_dim": 128, "rotated": 128, "interleaved": False, "page": 64, "past": 64, "heads_first": True},
        # the next token of one request, with the five most probable ones
        {"name": "logprobs_one", "path": "logprobs", "dtype": "float32", "rows": 1, "vocabulary": 32000, "top": 5, "scale": 1.0},
        # 64 requests over a large vocabulary, twenty alternatives each
        {"name": "logprobs_decode", "path": "logprobs", "dtype": "bfloat16", "rows": 64, "vocabulary": 131072, "top": 20, "scale": 1.0},
        # the tokens of answers that are scored: no alternatives
        {"name": "logprobs_score", "path": "logprobs", "dtype": "float32", "rows": 4096, "vocabulary": 32768, "top": 0, "scale": 1.25},
        # likewise over a vocabulary of odd size, with a few alternatives
        {"name": "logprobs_answers", "path": "logprobs", "dtype": "float16", "rows": 2048, "vocabulary": 150001, "top": 8, "scale": 1.0},
    ]


# ---- drawn cases -----------------------------------------------------------------------------------------------

def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice((1, 2, 4, 8))
    return kv * rng.choice((1, 1, 2, 4, 7, 8)), kv


def _draw_lora(rng):
    some = (lambda: _log(rng, 64, 8192)) if rng.random() < 0.3 else (lambda: max(16, _log(rng, 64, 8192) // 16 * 16))
    rows = _log(rng, 1, 8192)
    requests = rows if rows <= 128 and rng.random() < 0.6 else rng.randint(1, min(rows, 12))
    return {"path": "lora", "dtype": rng.choice(HALVES), "rows": rows, "N": some(), "K": some(),
            "rank": rng.choice((8, 16, 16, 32, 64, _log(rng, 1, 64))), "adapters": rng.randint(1, min(64, 2 * requests)),
            "requests": requests, "plain": rng.randint(0, requests // 3), "bias": rng.random() < 0.5}


def _draw_norm(rng):
    heads, kv_heads = _heads(rng)
    head_dim = rng.choice((64, 80, 96, 128, 256))
    return {"path": "norm", "dtype": rng.choice(HALVES), "tokens": _log(rng, 1, 16384), "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rotated": rng.choice((0, head_dim // 2, head_dim, head_dim)), "interleaved": rng.random() < 0.5,
            "furthest": _log(rng, 1 << 11, 1 << 20)}


def _draw_append(rng):
    heads, kv_heads = _heads(rng)
    head_dim, most = rng.choice((64, 80, 128)), 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    return {"path": "append", "dtype": rng.choice(HALVES), "batch": _log(rng, 1, 64), "most": most, "least": rng.randint(1, most),
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotated": rng.choice((head_dim // 2, head_dim)),
            "interleaved": rng.random() < 0.5, "page": rng.choice((16, 32, 64, 256)), "past": _log(rng, 1, 4096),
            "heads_first": rng.random() < 0.5}


def _draw_logprobs(rng):
    return {"path": "logprobs", "dtype": rng.choice(sorted(DTYPES)), "rows": _log(rng, 1, 4096), "vocabulary": _log(rng, 512, 200000),
            "top": rng.choice((0, 0, 1, 5, 8, 20, 32)), "scale": rng.choice((1.0, 1.0, 0.7, 1.25))}


def draw(rng):
    kinds = {"lora": _draw_lora, "norm": _draw_norm, "append": _draw_append, "logprobs": _draw_logprobs}
    path = rng.choice(sorted(kinds))
    most = [work(c) for c in listed() if c["path"] == path]
    while True:
        case = kinds[path](rng)
        w = work(case)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return case


# ---- work ------------------------------------------------------------------------------------------------------

def _spread(least, most, n):
    """n numbers from `most` down to `least`, evenly."""
    return [most - (most - least) * i // max(1, n - 1) for i in range(n)]


def _requests(case):
    """(adapter, rows) of each request: rows in uneven shares, -1 for requests without an adapter."""
    n, rows = case["requests"], case["rows"]
    weights = [2 + (5 * i) % 7 for i in range(n)]
    ends = [rows * sum(weights[:i + 1]) // sum(weights) for i in range(n)] if rows > n else list(range(1, n + 1))
    with_one = n - case["plain"]
    return [((i * 7) % case["adapters"] if i < with_one else -1, e - s) for i, (s, e) in enumerate(zip([0] + ends[:-1], ends))]


def work(case):
    if case["path"] == "lora":
        M, N, K, r = case["rows"], case["N"], case["K"], case["rank"]
        parts = [p for p in _requests(case) if p[0] >= 0 and p[1] > 0]
        used, turned = len({a for a, _ in parts}), sum(n for _, n in parts)
        return {"bytes": 2 * (M * K + N * K + M * N + used * r * (K + N) + N * case["bias"]) + 4 * (M + used),
                "flops": 2 * M * N * K + 2 * turned * r * (K + N)}
    if case["path"] == "norm":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 4 * n * case["head_dim"] + 8 * case["tokens"] + 2 * case["rotated"] + 4 * case["head_dim"],
                "flops": 4 * n * case["head_dim"] + 3 * n * case["rotated"]}
    if case["path"] == "append":
        n, H, C, D = sum(_spread(case["least"], case["most"], case["batch"])), case["heads"], case["kv_heads"], case["head_dim"]
        return {"bytes": 4 * n * (H + 2 * C) * D + 8 * case["batch"] + 4 * D, "flops": n * (H + C) * (4 * D + 3 * case["rotated"])}
    n = case["rows"] * case["vocabulary"]
    return {"bytes": n * (4 if case["dtype"] == "float32" else 2) + case["rows"] * (20 + 12 * case["top"]), "flops": 5 * n}


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

    s = {"path": case["path"]}
    if case["path"] == "lora":
        M, N, K, r, n = case["rows"], case["N"], case["K"], case["rank"], case["adapters"]
        parts = _requests(case)
        order = torch.randperm(n, device="cuda", generator=g, dtype=torch.int32)
        of = _ints([a for a, _ in parts])
        of = torch.where(of >= 0, order[of.clamp(min=0).long()], of)
        s.update(x=normal(M, K), w=normal(N, K, scale=K ** -0.5), lora_a=normal(n, r, K, scale=K ** -0.5),
                 lora_b=normal(n, N, r, scale=0.5 * r ** -0.5), scales=torch.rand(n, device="cuda", generator=g).add_(0.5),
                 adapters=of.repeat_interleave(_ints([p for _, p in parts])), bias=normal(N) if case["bias"] else None)
        return s
    if case["path"] == "logprobs":
        # a few tokens well above the rest; the given ones are mostly among the probable, one in 16 rows has none
        R, V = case["rows"], case["vocabulary"]
        logits = torch.empty(R, V, dtype=dtype, device="cuda")
        for first in range(0, R, 512):
            part = 2.0 * torch.randn(min(512, R - first), V, device="cuda", generator=g)
            logits[first:first + 512] = part + 0.02 * part.pow(3)
        some = torch.randint(0, V, (R, 8), device="cuda", generator=g)
        tokens = some.gather(1, logits.gather(1, some).float().argmax(1, keepdim=True))[:, 0]
        s.update(logits=logits, tokens=torch.where(torch.arange(R, device="cuda") % 16 == 15, -1, tokens), top=case["top"],
                 scale=case["scale"])
        return s
    H, C, D = case["heads"], case["kv_heads"], case["head_dim"]
    s.update(q_weight=normal(D, scale=0.2) + 1.0, k_weight=normal(D, scale=0.2) + 1.0, interleaved=case["interleaved"],
             freqs=_frequencies(case["rotated"]) if case["rotated"] else None)
    if case["path"] == "norm":
        # queries, keys and values as one projection leaves them
        qkv = normal(case["tokens"], H + 2 * C, D, scale=1.7)
        s.update(q=qkv[:, :H], k=qkv[:, H:H + C],
                 positions=torch.randint(0, case["furthest"], (case["tokens"],), device="cuda", generator=g))
        return s
    B, page = case["batch"], case["page"]
    new = _spread(case["least"], case["most"], B)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    past = [case["past"]] * B
    # pages dealt out of order
    held = [-(-(p + n) // page) for p, n in zip(past, new)]
    order = torch.randperm(sum(held) + 2, device="cuda", generator=g, dtype=torch.int32)
    table = torch.full((B, max(held)), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(max(held), device="cuda")[None, :] < torch.tensor(held, device="cuda")[:, None]] = order[:sum(held)]
    shape = (sum(held) + 2, C, page, D) if case["heads_first"] else (sum(held) + 2, page, C, D)
    k_cache, v_cache = normal(*shape), normal(*shape)
    qkv = normal(offsets[-1], H + 2 * C, D, scale=1.7)
    s.update(table=table, lengths=_ints(past), offsets=_ints(offsets) if case["most"] > 1 else None, new=new,
             k_cache=k_cache.transpose(1, 2) if case["heads_first"] else k_cache,
             v_cache=v_cache.transpose(1, 2) if case["heads_first"] else v_cache, q=qkv[:, :H], k=qkv[:, H:H + C], v=qkv[:, H + C:])
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------

def _plain_lora(s):
    x = s["x"].float()
    y = torch.matmul(x, s["w"].float().t())
    n, r, K = s["lora_a"].shape
    of, scales = s["adapters"], s["scales"]
    if x.shape[0] * r * max(K, y.shape[1]) <= 1 << 27:
        # every row with its own adapter
        mine = of.clamp(min=0).long()
        low = torch.matmul(s["lora_a"][mine].float(), x[:, :, None]) * torch.where(of < 0, 0.0, scales[mine])[:, None, None]
        y += torch.matmul(s["lora_b"][mine].float(), low)[:, :, 0]
    else:
        # every adapter with all rows, those of others left out
        for i in range(n):
            low = torch.matmul(x, s["lora_a"][i].float().t()) * torch.where(of == i, scales[i], 0.0)[:, None]
            y += torch.matmul(low, s["lora_b"][i].float().t())
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def _norm(x, weight):
    return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight.float()


def _rotate(x, positions, freqs, interleaved):
    """x [tokens, heads, dim] in 32 bits; the angles of far positions take 64."""
    if freqs is None:
        return x
    n = freqs.numel()
    angle = positions.double()[:, None] * freqs.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    one, two = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    a, b = one * cos - two * sin, two * cos + one * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _plain_norm(s, positions):
    return tuple(_rotate(_norm(x.float(), w), positions, s["freqs"], s["interleaved"]).to(x.dtype)
                 for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _plain_append(s):
    rows = torch.arange(s["q"].shape[0], device="cuda")
    if s["offsets"] is None:
        seq, place = rows, s["lengths"].long()
    else:
        seq = torch.searchsorted(s["offsets"], rows, right=True) - 1
        place = s["lengths"][seq] + rows - s["offsets"][seq]
    page = s["k_cache"].shape[1]
    at = s["table"][seq, place // page].long(), place % page
    q, k = _plain_norm(s, place)
    s["k_cache"][at] = k
    s["v_cache"][at] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_logprobs(s):
    R, V = s["logits"].shape
    parts, step = [], max(1, (1 << 27) // V)
    for first in range(0, R, step):
        # (zeros of both signs are one number)
        x, tokens = s["logits"][first:first + step].float() + 0.0, s["tokens"][first:first + step]
        given = tokens >= 0
        at = tokens.clamp(min=0)[:, None]
        d = (x - x.amax(1, keepdim=True)) * s["scale"]
        e = d.exp()
        total = e.sum(1, keepdim=True)
        entropy = total.log()[:, 0] - (e * d).sum(1) / total[:, 0]
        logprob = torch.where(given, (d.gather(1, at) - total.log())[:, 0], 0.0)
        mine, place = x.gather(1, at), torch.arange(V, device="cuda")
        rank = torch.where(given, ((x > mine) | ((x == mine) & (place < at))).sum(1), -1).int()
        # (ties go to the lowest token: whole numbers that order by value, then by token)
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * (1 << 32) + (V - 1 - place)
        best = V - 1 - (key.topk(s["top"], 1).values & 0xffffffff)
        parts.append((logprob, entropy, rank, d.gather(1, best) - total.log(), best.int()))
    return tuple(torch.cat(p) for p in zip(*parts))


def run(s):
    if own:
        from aitemplate_amd import eager

        if s["path"] == "lora":
            return eager.gemm_rcr_lora(s["x"], s["w"], s["lora_a"], s["lora_b"], s["adapters"], s["scales"], s["bias"])
        if s["path"] == "norm":
            return eager.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["freqs"], eps=EPS,
                                        interleaved=s["interleaved"])
        if s["path"] == "append":
            q = eager.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["offsets"], q=s["q"],
                                      freqs=s["freqs"], interleaved=s["interleaved"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                      eps=EPS)
            return q, s["k_cache"], s["v_cache"]
        return eager.token_logprobs(s["logits"], s["tokens"], top=s["top"], scale=s["scale"])
    if s["path"] == "lora":
        return _plain_lora(s)
    if s["path"] == "norm":
        return _plain_norm(s, s["positions"])
    return _plain_append(s) if s["path"] == "append" else _plain_logprobs(s)


# ---- what the operators are, in 64 bits ------------------------------------------------------------------------

def _exact_heads(x, weight, positions, freqs, interleaved):
    """Unit heads times sqrt(dims), then products of complex numbers."""
    x = x.double()
    length = (x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS
    y = x / length.sqrt() * weight.double()
    if freqs is None:
        return y
    n = freqs.numel()
    pairs = y[..., :2 * n].unflatten(-1, (n, 2)) if interleaved else y[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2)
    angle = positions.double().unsqueeze(-1) * freqs.double()
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle).unsqueeze(-2))
    y[..., :2 * n] = (turned if interleaved else turned.transpose(-1, -2)).reshape(*x.shape[:-1], 2 * n)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if s["path"] == "lora":
        x, y = s["x"].double(), torch.empty(case["rows"], case["N"], dtype=torch.float64, device="cuda")
        row = 0
        for _, n in _requests(case):
            # the request's own weight, its adapter added to the shared one
            w = s["w"].double()
            if n and int(s["adapters"][row]) >= 0:
                i = int(s["adapters"][row])
                w = w + s["scales"][i].double() * (s["lora_b"][i].double() @ s["lora_a"][i].double())
            y[row:row + n] = x[row:row + n] @ w.t()
            row += n
        return y if s["bias"] is None else y + s["bias"].double()
    if s["path"] == "norm":
        return tuple(_exact_heads(x, w, s["positions"], s["freqs"], s["interleaved"])
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    if s["path"] == "append":
        q, k, v = s["q"].double().clone(), s["k_cache"].double(), s["v_cache"].double()
        row, page = 0, s["k_cache"].shape[1]
        for b, n in enumerate(s["new"]):
            place = torch.arange(case["past"], case["past"] + n, device="cuda")
            at = s["table"][b, place // page].long(), place % page
            mine = slice(row, row + n)
            k[at] = _exact_heads(s["k"][mine], s["k_weight"], place, s["freqs"], s["interleaved"])
            q[mine] = _exact_heads(s["q"][mine], s["q_weight"], place, s["freqs"], s["interleaved"])
            v[at] = s["v"][mine].double()
            row += n
        return q, k, v
    logprob, entropy, best = [], [], []
    for first in range(0, case["rows"], 256):
        x, tokens = s["logits"][first:first + 256].double() * s["scale"], s["tokens"][first:first + 256]
        lp = torch.log_softmax(x, 1)
        logprob.append(lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0].masked_fill(tokens < 0, 0.0))
        entropy.append(-(lp.exp() * lp).sum(1))
        best.append(lp.topk(s["top"], 1).values)
    return torch.cat(logprob), torch.cat(entropy), None, torch.cat(best), None
