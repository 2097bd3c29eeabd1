"""Rotary positions on the GPU, against the rotation in 64 bits.

Tolerance: the result is rounded once (half a step of its type, eps / 2 relative).  Before that a pair (x1, x2) is off by at
most (|x1| + |x2|) * (the angle's 2 pi 2^-25 and the sines' 2^-22, under 5e-7; three roundings of 2^-24): 1e-6 covers both."""
import math

import pytest
import torch

from aitemplate_amd import eager

pytestmark = pytest.mark.gpu
DEV = "cuda"


def turned(x, positions, freqs, interleaved, scale=1.0, inverse=False):
    """The rotation in 64 bits, and the pairs' |x1| + |x2| laid out the same."""
    x = x.double()
    n = freqs.numel()
    angle = positions.double().unsqueeze(-1) * freqs.double()
    angle = (-angle if inverse else angle).unsqueeze(-2)
    y, size = x.clone(), torch.zeros_like(x)
    i1 = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    i2 = i1 + (1 if interleaved else n)
    a, b = x[..., i1], x[..., i2]
    y[..., i1] = scale * (a * angle.cos() - b * angle.sin())
    y[..., i2] = scale * (b * angle.cos() + a * angle.sin())
    size[..., i1] = size[..., i2] = (a.abs() + b.abs()) * abs(scale)
    return y, size


def check(got, x, positions, freqs, interleaved, scale=1.0, inverse=False):
    want, size = turned(x, positions, freqs, interleaved, scale, inverse)
    allowed = want.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 1e-4) + size * 1e-6 + torch.finfo(got.dtype).smallest_normal
    worst = ((got.double() - want).abs() / allowed).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst


def freqs_of(rotated):
    return eager.rotary_frequencies(rotated, device=DEV)[0] if rotated else torch.empty(0, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,head_dim,rotated", [
    (1, 1, 2, 2), (1, 32, 128, 128), (7, 12, 64, 64), (33, 3, 80, 40), (130, 5, 96, 48), (5, 7, 72, 16), (1000, 1, 64, 32),
    (9, 4, 10, 6), (3, 2, 129, 30), (2, 71, 64, 0), (4, 2, 1024, 1024), (700, 16, 256, 256), (3, 2, 24, 12)])
def test_rotation(dtype, interleaved, tokens, heads, head_dim, rotated):
    g = torch.Generator(device=DEV).manual_seed(tokens + head_dim)
    x = torch.randn(tokens, heads, head_dim, device=DEV, generator=g).to(dtype)
    positions = torch.randint(0, 1 << 20, (tokens,), device=DEV, generator=g)
    freqs = freqs_of(rotated)
    check(eager.rotary_embedding(x, positions, freqs, interleaved), x, positions, freqs, interleaved)
    got = eager.rotary_embedding(x, positions.int(), freqs, interleaved, scale=1.25, inverse=True)
    check(got, x, positions, freqs, interleaved, 1.25, True)


@pytest.mark.parametrize("far", [0, -5, (1 << 31) - 1, 1 << 40])
def test_far_positions(far):
    x = torch.randn(3, 2, 64, device=DEV).half()
    positions = torch.tensor([far, far - 1, far + 1], device=DEV)
    freqs = freqs_of(64)
    # (beyond 2^31 the oracle's own angle, position * frequency in 64 bits, is off by up to 2^41 * 2^-53 = 2^-12)
    if abs(far) > 1 << 31:
        turns = torch.remainder(positions.double(), 2.0 * math.pi)
        freqs = torch.ones(32, device=DEV)
        want, _ = turned(x, turns, freqs, False)
        assert (eager.rotary_embedding(x, positions, freqs).double() - want).abs().max().item() < 2e-2
        return
    want, size = turned(x, positions, freqs, False)
    allowed = want.abs() * 2.0 ** -11 * (1 + 1e-4) + size * (1e-6 + abs(far) * 2.0 ** -51) + 2.0 ** -14
    assert ((eager.rotary_embedding(x, positions, freqs).double() - want).abs() <= allowed).all()


def test_more_tokens_than_one_launch_takes():
    # (2^24 workgroups of 64 tokens and two more)
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of free memory")
    x = torch.ones((1 << 30) + 70, 1, 2, dtype=torch.float16, device=DEV)
    positions = torch.zeros(x.shape[0], dtype=torch.int32, device=DEV)
    assert eager.rotary_embedding(x, positions, freqs_of(2), scale=2.0, out=x) is x
    assert (x == 2).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strides_batches_and_places(dtype):
    B, S, H, D = 3, 17, 4, 64
    freqs = freqs_of(D)
    qkv = torch.randn(B, S, 3 * H, D, device=DEV).to(dtype)
    before = qkv.clone()
    q = qkv[:, :, H:2 * H]
    one_row = torch.arange(S, device=DEV) + 100
    per_entry = torch.randint(0, 4096, (B, S), device=DEV)
    for positions in (one_row, per_entry, per_entry.t().contiguous().t()):
        each = positions.expand(B, S)
        check(eager.rotary_embedding(q, positions, freqs), q, each, freqs, False)
        # heads ahead of the sequence, as the attention ops take them
        out = torch.empty(B, H, S, D, device=DEV, dtype=dtype)
        eager.rotary_embedding(q, positions, freqs, out=out.transpose(1, 2))
        check(out.transpose(1, 2), q, each, freqs, False)
    # in place, and nothing beside it touched
    want = eager.rotary_embedding(q, one_row, freqs)
    assert eager.rotary_embedding(q, one_row, freqs, out=q) is q
    assert torch.equal(q, want)
    assert torch.equal(qkv[:, :, :H], before[:, :, :H]) and torch.equal(qkv[:, :, 2 * H:], before[:, :, 2 * H:])
    # elements at any address
    odd = torch.randn(1 + 5 * H * D, device=DEV).to(dtype)[1:].view(5, H, D)
    check(eager.rotary_embedding(odd, one_row[:5], freqs, True), odd, one_row[:5], freqs, True)


def test_there_and_back_and_gradient():
    x = torch.randn(11, 3, 48, device=DEV).bfloat16()
    dy = torch.randn(11, 3, 48, device=DEV).bfloat16()
    positions, freqs = torch.arange(11, device=DEV) * 1000, freqs_of(32)
    for interleaved in (False, True):
        back = eager.rotary_embedding(eager.rotary_embedding(x, positions, freqs, interleaved), positions, freqs, interleaved, inverse=True)
        # two roundings, each of a value of at most sqrt(2) times the pair's larger one
        assert ((back - x).double().abs() <= 2.0 ** -7 * 3 * x.abs().max().double()).all()
        # <dy, R(x)> has the gradient R^T dy: by differences in 64 bits, exact as the operator is linear
        grad = eager.rotary_embedding(dy, positions, freqs, interleaved, scale=1.5, inverse=True).double()
        step = torch.randn(11, 3, 48, device=DEV).double()
        ahead, size = turned(x.double() + step, positions, freqs, interleaved, 1.5)
        behind, _ = turned(x.double() - step, positions, freqs, interleaved, 1.5)
        along = (dy.double() * (ahead - behind)).sum() / 2
        allowed = (grad.abs() * step.abs()).sum() * 2.0 ** -8 + (dy.double().abs() * step.abs()).sum() * 1e-5
        assert (along - (grad * step).sum()).abs() <= allowed


def test_infinities_and_nan_stay_in_their_pairs():
    x = torch.randn(2, 2, 64, device=DEV).half()
    x[0, 0, 3], x[1, 1, 40] = math.inf, math.nan
    positions, freqs = torch.tensor([5, 6], device=DEV), freqs_of(64)
    y = eager.rotary_embedding(x, positions, freqs)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, 3] = want[0, 0, 35] = want[1, 1, 40] = want[1, 1, 8] = True
    assert torch.equal(bad, want)


def test_captured_and_replayed():
    x = torch.randn(64, 8, 128, device=DEV).half()
    positions, freqs = torch.arange(64, device=DEV), freqs_of(128)
    out = torch.empty_like(x)
    eager.rotary_embedding(x, positions, freqs, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eager.rotary_embedding(x, positions, freqs, out=out)
    for k in range(4):
        x.normal_()
        positions += 7
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager.rotary_embedding(x, positions, freqs))
