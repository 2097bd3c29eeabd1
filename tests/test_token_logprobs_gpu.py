"""Log probabilities, entropies, ranks and alternatives on the GPU, against 64 bits.

Tolerance: the sum of V positive numbers in 32 bits, V / 512 of them a thread and then some 60 joined (up to 32 parts of 512 threads,
with a multiplication each), is off by at most (V / 512 + 128) 2^-24 of itself, its exponentials by 2^-21 (the last bits of a
distance d of up to 40 that counts, and the instruction's); both enter the logarithm as they are.  The distances themselves: 2^-22 of
the log probability and of ln V.  The entropy has the mean distance, off likewise, besides."""
import math

import pytest
import torch

from aitemplate_amd import eager

pytestmark = pytest.mark.gpu
DEV = "cuda"


def order(logits):
    """Tokens by logit, then by index; NaN last."""
    x = logits.double().nan_to_num(nan=-float("inf"), posinf=float("inf"), neginf=-float("inf"))
    last = torch.where(logits.isnan(), 1, 0)
    by_value = torch.sort(x, dim=-1, descending=True, stable=True).indices
    return by_value.gather(-1, torch.sort(last.gather(-1, by_value), dim=-1, stable=True).indices)


def check(got, logits, tokens, top=0, scale=1.0):
    logprob, entropy, rank, top_logprob, top_token = got
    V = logits.shape[-1]
    lp = torch.log_softmax(logits.double() * scale, -1)
    p_lp = torch.where(lp == -float("inf"), 0.0, lp.exp() * lp)
    want_entropy = -p_lp.sum(-1)
    given = (tokens >= 0) & (tokens < V)
    want = torch.where(given, lp.gather(-1, tokens.clamp(0, V - 1).long().unsqueeze(-1)).squeeze(-1), 0.0)
    sums = (V / 512 + 128) * 2.0 ** -24 + 2.0 ** -21

    def close(a, b, off):
        same = (a.double() == b) | ((a.double() - b).abs() <= off)
        assert same.all(), ((a.double() - b).abs() / off).max().item()

    size = math.log(V) + 2.0
    close(logprob, want, sums + 2.0 ** -22 * (want.abs().nan_to_num(posinf=0.0) + size))
    mean = (-(lp.amax(-1)) - want_entropy).abs() + size  # (of the distances, and ln of the sum)
    close(entropy, want_entropy, (2 * sums + 2.0 ** -21) * (mean + 1))
    places = order(logits)
    of = (places == tokens.clamp(0, V - 1).long().unsqueeze(-1)).int().argmax(-1)
    assert torch.equal(rank.long(), torch.where(given, of, -1))
    assert top_token.shape == logits.shape[:-1] + (top,) and torch.equal(top_token.long(), places[..., :top])
    best = lp.gather(-1, places[..., :top])
    close(top_logprob, best, sums + 2.0 ** -22 * (best.abs().nan_to_num(posinf=0.0) + size))


def make(dtype, rows, V, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = (torch.randn(rows, V, device=DEV, generator=g) * spread).to(dtype)
    tokens = torch.randint(0, V, (rows,), device=DEV, generator=g)
    tokens[::7] = -1
    return logits, tokens


DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (1, 2, 2), (3, 7, 7), (5, 64, 64), (2, 511, 20), (1, 4096, 5), (4, 8191, 33), (1, 8192, 1),
                                        (3, 8193, 64), (2, 40000, 20), (1, 150001, 8), (700, 1000, 0), (600, 3001, 4), (1030, 20000, 20),
                                        (1, 300000, 64)])
def test_rows(dtype, rows, V, top):
    logits, tokens = make(dtype, rows, V, seed=rows + V)
    for scale in (1.0, 0.7):
        check(eager.token_logprobs(logits, tokens, top=top, scale=scale), logits, tokens, top, scale)
    check(eager.token_logprobs(logits, tokens.int()), logits, tokens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("shape", ["ascending", "descending", "equal", "few values", "one apart", "steps of a thread"])
def test_orders(dtype, rows, shape):
    """Rows whose candidates do not fit at once, and ties."""
    V = 30011
    at = torch.arange(V, device=DEV)
    row = {"ascending": at / V * 8 - 4, "descending": 4 - at / V * 8, "equal": torch.full((V,), 1.5, device=DEV), "few values": (at * 7919 % 5).float(),
           "one apart": torch.where(at == V - 3, 9.0, 0.0), "steps of a thread": (at // 8 % 512).float() * 0.02 + at / V * 0.01}[shape]
    logits = row.to(dtype).expand(rows, V).contiguous()
    tokens = torch.arange(rows, device=DEV) * 41 % V
    for top in (1, 20, 64):
        check(eager.token_logprobs(logits, tokens, top=top), logits, tokens, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 530])
def test_masked(dtype, rows):
    logits, tokens = make(dtype, rows, 9001, seed=1)
    low = torch.finfo(dtype).min
    logits[:, 5:8000] = -float("inf")
    check(eager.token_logprobs(logits, tokens, top=20), logits, tokens, 20)
    logits[:, 5:8990] = low
    check(eager.token_logprobs(logits, tokens, top=20), logits, tokens, 20)
    # rows of nothing but the lowest number are even ones
    logits.fill_(low)
    check(eager.token_logprobs(logits, tokens, top=3), logits, tokens, 3)
    # one token left; none
    logits.fill_(-float("inf"))
    logits[:, 4321] = 0.5
    tokens[0] = 4321
    check(eager.token_logprobs(logits, tokens, top=3), logits, tokens, 3)
    logits.fill_(-float("inf"))
    logprob, entropy, rank, top_logprob, top_token = eager.token_logprobs(logits, tokens, top=3)
    given = tokens >= 0
    assert (logprob[given] == -float("inf")).all() and (logprob[~given] == 0).all() and (entropy == 0).all()
    assert (top_logprob == -float("inf")).all() and (top_token == torch.arange(3, device=DEV)).all()
    assert torch.equal(rank.long(), torch.where(given, tokens, -1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_numbers(dtype):
    logits, tokens = make(dtype, 5, 20001, seed=2)
    tokens[:] = 17
    logits[1, 19000], logits[2, 3], logits[3] = float("inf"), float("nan"), float("nan")
    logits[3, 40] = 1.0
    logprob, entropy, rank, top_logprob, top_token = eager.token_logprobs(logits, tokens, top=4)
    ordinary = [0, 4]
    check([t[ordinary] for t in (logprob, entropy, rank, top_logprob, top_token)], logits[ordinary], tokens[ordinary], 4)
    assert logprob[1:4].isnan().all() and entropy[1:4].isnan().all()
    assert torch.equal(top_token[1:3].long(), order(logits[1:3])[:, :4])
    assert top_token[3].tolist() == [40, -1, -1, -1]


def test_zeros_of_both_signs_are_one_number():
    logits = torch.zeros(1, 100, device=DEV)
    logits[0, ::2] = -0.0
    tokens = torch.tensor([50], device=DEV)
    check(eager.token_logprobs(logits, tokens, top=10), logits.abs(), tokens, 10)


def test_pitch_leading_dims_and_tokens_out_of_range():
    logits, tokens = make(torch.bfloat16, 6, 5003, seed=3)
    wide = torch.full((6, 6001), float("nan"), device=DEV).bfloat16()
    wide[:, 7:5010] = logits
    check(eager.token_logprobs(wide[:, 7:5010], tokens, top=5), logits, tokens, 5)
    got = eager.token_logprobs(logits.view(2, 3, 5003), tokens.view(2, 3), top=5)
    check(got, logits.view(2, 3, 5003), tokens.view(2, 3), 5)
    tokens[:4] = torch.tensor([5003, -7, 1 << 40, 5002], device=DEV)
    check(eager.token_logprobs(logits, tokens), logits, tokens)


def test_empty():
    got = eager.token_logprobs(torch.empty(0, 50, device=DEV), torch.empty(0, dtype=torch.long, device=DEV), top=3)
    assert [t.shape for t in got] == [(0,), (0,), (0,), (0, 3), (0, 3)]


def test_the_same_twice_and_captured():
    logits, tokens = make(torch.float16, 8, 60000, seed=4)
    logits = (logits * 4).round() / 4  # (many equal ones)
    need = eager.token_logprobs_workspace_bytes(8, 60000, 20)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = eager.token_logprobs(logits, tokens, top=20, workspace=ws)
    for step in range(4):
        logits.copy_((torch.randn_like(logits) * 12).round() / 4)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, eager.token_logprobs(logits, tokens, top=20)):
            assert torch.equal(a, b)


def test_refusals():
    logits, tokens = make(torch.float16, 4, 100)
    for args, word in (((logits.double(), tokens), "logits"), ((logits, tokens.float()), "tokens"), ((logits, tokens[:3]), "tokens"),
                       ((logits.t(), tokens), "contiguous"), ((logits, tokens.cpu()), "tokens")):
        with pytest.raises(ValueError, match=word):
            eager.token_logprobs(*args)
    for kw, word in ((dict(top=65), "top"), (dict(top=-1), "top"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")):
        with pytest.raises(RuntimeError, match=word):
            eager.token_logprobs(logits, tokens, **kw)
    with pytest.raises(RuntimeError, match="top"):
        eager.token_logprobs(logits[:, :10], tokens, top=11)
    big, t = make(torch.float16, 1, 50000)
    with pytest.raises(RuntimeError, match="workspace"):
        eager.token_logprobs(big, t, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
