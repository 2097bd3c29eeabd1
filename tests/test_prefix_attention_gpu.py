"""Attention over a paged cache with a shared prefix on the GPU, against the formula in 64 bits.

Tolerance, with eps the type's step, w the weights, A = sum w |v| and y the result: the weights are taken as rounded
probabilities over the sum of the rounded ones, each off by eps / 2 at most, which moves y by eps / 2 (A + |y|); the result is
rounded once, eps / 2 |y|.  A score is a sum of D products in 32 bits, off by at most D 2^-24 sum |q k| scale, an exponential by
2^-22 more; twice that, relative, moves y by as much of A + |y|.  In fp16 a probability below 2^-14 is off by 2^-25 at most
instead, against a sum of at least 1: n 2^-25 max |v| for n keys.  The sums of up to n products in 32 bits: sqrt would do, n 2^-24
A is certain, 2^-14 A at most here."""
import math

import pytest
import torch

from aitemplate_amd import eager
from paged_common import DEV, Paged

pytestmark = pytest.mark.gpu


def one_sequence(q, k, v, hidden, scale, dtype):
    """(result, allowed error) of rows q [n, heads, D] over keys k, v [N, kv_heads, D]; hidden [n, N]."""
    H, C = q.shape[1], k.shape[1]
    if k.shape[0] == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    q, k, v = (t.double().transpose(0, 1) for t in (q, k.repeat_interleave(H // C, 1), v.repeat_interleave(H // C, 1)))
    score = (q @ k.transpose(1, 2).contiguous()) * scale
    size = (q.abs() @ k.abs().transpose(1, 2).contiguous()) * abs(scale)
    score = score.masked_fill(hidden, -math.inf)
    w = torch.softmax(score, -1).nan_to_num(0.0)
    v = v.contiguous()
    y, a = w @ v, w @ v.abs()
    off = (size.masked_fill(hidden, 0.0).amax(-1, keepdim=True) * q.shape[2] * 2.0 ** -24 + 2.0 ** -22) * 2
    eps = torch.finfo(dtype).eps / 2
    small = k.shape[1] * 2.0 ** -25 * v.abs().amax() if dtype == torch.float16 else 0.0
    allowed = (eps + off) * 1.01 * (a + y.abs()) + eps * y.abs() + 2.0 ** -14 * a + small + torch.finfo(dtype).smallest_normal
    return y.transpose(0, 1), allowed.transpose(0, 1)


def operands(c, heads, kv_heads, head_dim, strided=False):
    rows = torch.randn(c.tokens, heads + 2 * kv_heads, head_dim, device=DEV).to(c.dtype)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    for i in range(len(c.past)):
        mine, at = slice(c.starts[i], c.starts[i + 1]), c.past[i]
        skip = max(0, -at)
        c.fill(c.k, c.table[i], max(0, at), k[mine][skip:])
        c.fill(c.v, c.table[i], max(0, at), v[mine][skip:])
    return q if strided else q.contiguous()


def check(c, q, got, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    shared = [c.read(t, c.prefix_table, c.prefix) for t in (c.k, c.v)]
    worst = 0.0
    for i, (p, n) in enumerate(zip(c.past, c.new)):
        if n == 0:
            continue
        own = [c.read(t, c.table[i], p + n) for t in (c.k, c.v)]
        k, v = (torch.cat(pair) for pair in zip(shared, own))
        hidden = torch.arange(k.shape[0], device=DEV) >= c.prefix + torch.arange(p + 1, p + n + 1, device=DEV)[:, None].clamp(min=0)
        rows = slice(c.starts[i], c.starts[i + 1])
        want, allowed = one_sequence(q[rows], k, v, hidden, scale, c.dtype)
        off = (got[rows].double() - want).abs()
        assert torch.isfinite(got[rows]).all(), i
        assert (off <= allowed).all(), (i, (off / allowed).nan_to_num(0.0).max().item())
        worst = max(worst, (off / allowed).nan_to_num(0.0).max().item())
    return worst


def attend(c, q, **more):
    return eager.prefix_attention(q, c.k, c.v, c.table, c.lengths, c.offsets, prefix_table=c.prefix_table if c.prefix else None,
                                  prefix_length=c.prefix, **more)


ONE_TOKEN = [
    # past, heads, kv_heads, head_dim, page, prefix
    ([0], 1, 1, 64, 16, 0),
    ([0], 1, 1, 8, 16, 1),
    ([61], 12, 12, 64, 16, 384),
    ([0, 15, 16, 17, 127, 128, 129, 1000], 8, 2, 128, 16, 0),
    ([0, 15, 16, 17, 127, 128, 129, 1000], 8, 2, 128, 16, 777),
    (list(range(0, 700, 10)), 8, 1, 96, 32, 65),
    ([300, 0, 40], 40, 1, 80, 48, 130),     # more query heads than a row tile has rows
    ([300, 7], 71, 1, 64, 16, 0),
    ([513, 100, 31], 7, 7, 72, 256, 15),
    ([513, 100, 31], 6, 3, 160, 16, 16),
    ([513, 100, 31], 4, 2, 256, 64, 2041),
    ([5000], 4, 1, 128, 16, 0),             # one sequence, its keys shared between workgroups
    ([3], 4, 1, 128, 16, 9000),
    ([20000, 3], 4, 1, 64, 16, 20000),      # as many parts of a row as the join takes
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("past,heads,kv_heads,head_dim,page,prefix", ONE_TOKEN)
def test_one_token(dtype, heads_first, past, heads, kv_heads, head_dim, page, prefix):
    c = Paged(dtype, past, [1] * len(past), kv_heads, head_dim, page, prefix, heads_first)
    q = operands(c, heads, kv_heads, head_dim, strided=True)
    check(c, q, attend(c, q))


RAGGED = [
    # past, new, heads, kv_heads, head_dim, page, prefix
    ([0, 5, 7, 31], [1, 2, 0, 3], 8, 2, 64, 16, 100),
    ([0, 0, 0], [0, 0, 1], 4, 4, 128, 16, 0),
    ([3, 0, 40], [50, 170, 10], 6, 3, 80, 16, 0),
    ([0, 50, 64, 31], [127, 128, 129, 1], 4, 4, 64, 64, 63),
    ([1333, 0, 700], [5, 517, 260], 16, 4, 80, 64, 2041),
    ([10, 0], [300, 257], 5, 1, 256, 32, 17),
    ([0], [1000], 2, 2, 96, 16, 0),
    ([100], [40], 8, 8, 128, 16, 3000),
    ([i % 9 for i in range(150)], [(3 * i) % 5 for i in range(150)], 4, 1, 64, 16, 33),
    ([i % 9 for i in range(150)], [(7 * i) % 90 for i in range(150)], 2, 1, 64, 16, 33),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("past,new,heads,kv_heads,head_dim,page,prefix", RAGGED)
def test_ragged(dtype, heads_first, past, new, heads, kv_heads, head_dim, page, prefix):
    c = Paged(dtype, past, new, kv_heads, head_dim, page, prefix, heads_first, ragged=True)
    q = operands(c, heads, kv_heads, head_dim)
    check(c, q, attend(c, q))


def test_scores_of_any_size_and_scale():
    for dtype in (torch.float16, torch.bfloat16):
        c = Paged(dtype, [700, 20], [1, 1], 2, 64, 16, 500)
        q = operands(c, 8, 2, 64)
        for scale in (1.0, -0.3, 0.0, 20.0):
            check(c, q, attend(c, q, scale=scale), scale)
        # a maximum that grows from tile to tile
        grows = torch.arange(700, device=DEV).double() / 60
        own = c.table[0][torch.arange(700, device=DEV) // 16].long(), torch.arange(700, device=DEV) % 16
        c.k[own] = (c.k[own].double() * grows[:, None, None]).to(dtype)
        check(c, q, attend(c, q, scale=1.0), 1.0)


def test_rows_without_a_key_and_sequences_that_are_not_there():
    for prefix in (0, 40):
        # lengths below zero: the first rows see no key of their own
        c = Paged(torch.float16, [-1, 4, -3, -2], [1, 1, 6, 2], 2, 64, 16, prefix)
        q = operands(c, 4, 2, 64)
        got = attend(c, q)
        check(c, q, got)
        if not prefix:
            assert not got[0].any() and not got[2:4].any() and not got[8:].any() and got[4:8].any()
        c = Paged(torch.bfloat16, [-1, 4, -1000], [1, 1, 1], 2, 64, 16, prefix)
        q = operands(c, 4, 2, 64)
        check(c, q, attend(c, q))


def test_no_table_at_all():
    c = Paged(torch.float16, [0, 0], [1, 1], 2, 64, 16, 50)
    q = operands(c, 4, 2, 64)
    c.table = c.table[:, :0]
    got = attend(c, q)
    keys = [c.read(t, c.prefix_table, 50) for t in (c.k, c.v)]
    want, allowed = one_sequence(q, *keys, torch.zeros(2, 50, dtype=torch.bool, device=DEV), 0.125, torch.float16)
    assert ((got.double() - want).abs() <= allowed).all()


def test_rows_of_nobody_stay_and_pages_outside_count_as_zeros():
    c = Paged(torch.float16, [20, 3], [2, 4], 2, 64, 16, 33)
    operands(c, 4, 2, 64)
    q = torch.randn(11, 4, 64, device=DEV).half()
    out = torch.full((11, 4, 64), 9.0, device=DEV, dtype=torch.float16)
    assert attend(c, q, out=out) is out
    check(c, q, out)
    assert (out[6:] == 9.0).all()
    # the second page of sequence 0 (its keys 16 to 21) is none
    for none in (-1, c.k.shape[0], 1 << 30):
        gone = c.table[0, 1].item()
        c.table[0, 1] = none
        got = attend(c, q)[:6]
        c.table[0, 1] = gone
        held = [t[gone].clone() for t in (c.k, c.v)]
        c.k[gone], c.v[gone] = 0.0, 0.0
        check(c, q, got)
        c.k[gone], c.v[gone] = held


def test_infinities_and_nan():
    c = Paged(torch.float16, [40, 40, 40], [1, 1, 1], 1, 64, 16, 20)
    q = operands(c, 2, 1, 64)
    clean = attend(c, q)
    # one sequence's NaN is its own; so is an infinity; a query's NaN is its row's
    c.v[c.table[0, 1].long(), 3, 0, 5] = math.nan
    c.v[c.table[1, 0].long(), 2, 0, 7] = math.inf
    q[2, 1, 9] = math.nan
    got = attend(c, q)
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, :, 5] = want[1, :, 7] = want[2, 1, :] = True
    assert torch.equal(bad, want) and torch.isinf(got[1, :, 7]).all()
    assert torch.equal(got[~bad], clean[~bad])


def test_a_later_rows_key_may_be_anything():
    # a key that only later rows of the step see is masked for the others, NaN and infinities too
    c = Paged(torch.bfloat16, [10], [40], 1, 64, 16)
    q = operands(c, 4, 1, 64)
    clean = attend(c, q)
    place = 10 + 30
    c.k[c.table[0, place // 16].long(), place % 16, 0, 5] = math.nan
    got = attend(c, q)
    assert torch.equal(got[:30], clean[:30]) and torch.isnan(got[30:]).all()


def test_offsets_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of free memory")
    D, stride = 64, 1 << 29
    k_all, v_all = (torch.empty(5 * (1 << 30) // 2 + 16 * D, dtype=torch.float16, device=DEV) for _ in range(2))
    c = Paged(torch.float16, [15], [1], 1, D, 16)
    q = operands(c, 4, 1, D)
    k, v = (t.as_strided((5, 16, 1, D), (stride, D, D, 1)) for t in (k_all, v_all))
    k[4], v[4] = c.k[c.table[0, 0].long()], c.v[c.table[0, 0].long()]
    table = torch.tensor([[4]], dtype=torch.int32, device=DEV)
    assert torch.equal(eager.prefix_attention(q, k, v, table, c.lengths), attend(c, q))


def test_on_another_stream_with_a_workspace_and_the_same_each_time():
    c = Paged(torch.float16, [3000, 10], [1, 1], 2, 128, 16, 1000)
    q = operands(c, 8, 2, 128)
    want = attend(c, q)
    need = eager.prefix_attention_workspace_bytes(q, c.k, c.v, c.table, c.lengths, prefix_length=1000)
    assert need > 0
    workspace = torch.full((need,), 255, dtype=torch.uint8, device=DEV)  # NaN
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [attend(c, q, workspace=workspace) for _ in range(3)]
    stream.synchronize()
    assert all(torch.equal(g, want) for g in got)
    with pytest.raises(RuntimeError, match="workspace"):
        attend(c, q, workspace=workspace[:-1].clone())


def test_captured_and_replayed_while_lengths_grow():
    c = Paged(torch.bfloat16, [30, 14, 0], [1, 1, 1], 2, 64, 16, 50, spare=10)
    c.table = torch.cat((c.table, torch.full((3, 3), -1, dtype=torch.int32, device=DEV)), 1).contiguous()
    spare = iter(c.spare.tolist())
    held = [-(-(p + 1) // 16) for p in c.past]
    lengths = c.lengths.clone()
    q, out = torch.randn(3, 4, 64, device=DEV).bfloat16(), torch.empty(3, 4, 64, device=DEV, dtype=torch.bfloat16)

    def step(out):
        return eager.prefix_attention(q, c.k, c.v, c.table, lengths, prefix_table=c.prefix_table, prefix_length=50, out=out)

    operands(c, 4, 2, 64)
    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for _ in range(5):
        for i in range(3):
            if c.past[i] + 1 > held[i] * 16:
                c.table[i, held[i]] = next(spare)
                held[i] += 1
        operands(c, 4, 2, 64)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(torch.empty_like(out)))
        check(c, q, out)
        lengths += 1
        c.past = [p + 1 for p in c.past]
        for i in range(3):
            if c.past[i] + 1 > held[i] * 16:
                c.table[i, held[i]] = next(spare)
                held[i] += 1
