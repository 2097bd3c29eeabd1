"""Heads normalized and rotated on the GPU, by themselves and on their way into a paged cache, against 64 bits.

Tolerance: the result is rounded once (half a step of its type, eps / 2 relative).  Before that a number is off by at most (dim / 2 + 8)
2^-24 of itself: the squares' sum in 32 bits, under the root, and the roundings of the products; and the rotation adds 1e-6 of its
pair's magnitudes (see test_rotary_gpu.py)."""
import pytest
import torch

from aitemplate_amd import eager
from paged_common import DEV, Paged
from test_rotary_gpu import freqs_of, turned

pytestmark = pytest.mark.gpu


def normed(x, weight, eps):
    x = x.double()
    if weight is None:
        return x
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return torch.where(x == 0, x, x * r) * weight.double()


def check(got, x, weight, positions, freqs, eps=1e-6, interleaved=False, scale=1.0):
    v = normed(x, weight, eps)
    freqs = freqs_of(0) if freqs is None else freqs
    want, size = turned(v, positions, freqs, interleaved, scale)
    size = torch.where(size == 0, want.abs(), size)
    info = torch.finfo(got.dtype)
    allowed = want.abs() * info.eps / 2 * (1 + 1e-4) + size * (1e-6 + (x.shape[-1] / 2 + 8) * 2.0 ** -24) + info.smallest_normal * info.eps
    worst = ((got.double() - want).abs() / allowed).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,rotated", [
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 12, 4, 64, 64), (33, 3, 1, 80, 40), (130, 5, 5, 96, 48), (5, 7, 7, 72, 16), (1000, 2, 1, 64, 32),
    (9, 4, 2, 10, 6), (3, 2, 1, 129, 30), (2, 71, 3, 64, 0), (4, 2, 2, 1024, 1024), (700, 16, 4, 256, 128), (3, 2, 1, 24, 12),
    (5, 3, 1, 1024, 0), (2, 1, 3, 1023, 10), (3, 2, 2, 1, 0)])
def test_heads(dtype, interleaved, tokens, heads, kv_heads, head_dim, rotated):
    g = torch.Generator(device=DEV).manual_seed(tokens + head_dim)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    qkv = normal(tokens, heads + 2 * kv_heads, head_dim) * 3
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv_heads]
    positions = torch.randint(0, 1 << 20, (tokens,), device=DEV, generator=g)
    freqs = freqs_of(rotated) if rotated else None
    qw, kw = normal(head_dim), normal(kv_heads, head_dim)
    got = eager.qk_norm_rotary(q, k, qw, kw, positions, freqs, interleaved=interleaved)
    check(got[0], q, qw, positions, freqs, interleaved=interleaved)
    check(got[1], k, kw, positions, freqs, interleaved=interleaved)
    # keys alone of other weights, an eps that counts, in place; queries rotated only
    mine = qkv.clone()
    out = eager.qk_norm_rotary(mine[:, :heads], mine[:, heads:heads + kv_heads], None, kw[0], positions.int(), freqs, eps=0.5,
                               interleaved=interleaved, scale=1.25, q_out=mine[:, :heads], k_out=mine[:, heads:heads + kv_heads])
    assert out[0].data_ptr() == mine.data_ptr()
    check(mine[:, :heads], q, None, positions, freqs, interleaved=interleaved, scale=1.25)
    check(mine[:, heads:heads + kv_heads], k, kw[0], positions, freqs, 0.5, interleaved, 1.25)
    assert torch.equal(mine[:, heads + kv_heads:], qkv[:, heads + kv_heads:])


def test_batches_and_strides():
    x = torch.randn(3, 5, 6, 64, device=DEV).half()
    k = torch.randn(6, 3, 5, 80, device=DEV).half().permute(1, 2, 0, 3)[:, :, :2, 4:68]
    w = torch.randn(6, 64, device=DEV).half()
    freqs = freqs_of(64)
    for positions in (torch.arange(5, device=DEV), torch.randint(0, 99, (3, 10), device=DEV)[:, ::2]):
        q_out = torch.zeros(3, 6, 5, 64, device=DEV).half().transpose(1, 2)
        got = eager.qk_norm_rotary(x, k, w, w[0], positions, freqs, q_out=q_out)
        check(got[0], x, w, positions.expand(3, 5), freqs)
        check(got[1], k, w[0], positions.expand(3, 5), freqs)
    alone, none = eager.qk_norm_rotary(x, None, w, None, positions, freqs)
    assert none is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head_dim", [64, 1024])
def test_heads_of_any_size(dtype, head_dim):
    """Zeros, with eps and without, squares that leave 32 bits, infinities and NaN beside ordinary heads."""
    x = torch.randn(8, 2, head_dim, device=DEV).to(dtype)
    w, positions = torch.ones(head_dim, device=DEV).to(dtype), torch.arange(8, device=DEV)
    big, small = (1e38, 1e-38) if dtype is torch.bfloat16 else (6e4, 6e-8)
    x[0] = 0
    x[1] = x[1].sign() * big
    x[2] = x[2].sign() * small
    x[3, 0, 5], x[4, 0, 5] = float("inf"), float("nan")
    for eps in (0.0, 1e-6):
        y = eager.qk_norm_rotary(x, None, w, None, positions, None, eps=eps)[0]
        ordinary = [0, 1, 2, 5, 6, 7]
        check(y[ordinary], x[ordinary], w, positions[ordinary], None, eps)
        assert (y[0] == 0).all() and y[4, 0].isnan().all()
        rest = torch.arange(head_dim, device=DEV) != 5
        assert y[3, 0, 5].isnan() and (y[3, 0, rest] == 0).all()
        check(y[3:5, 1:], x[3:5, 1:], w, positions[3:5], None, eps)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("past,new,heads,kv_heads,head_dim,rotated,page,heads_first", [
    ([5], [1], 4, 4, 64, 64, 16, False), ([20, 3, 40, 0], [1, 1, 1, 1], 8, 2, 128, 128, 16, True), ([0, 31, 7], [33, 1, 20], 6, 3, 80, 40, 16, False),
    ([100, 0], [7, 0], 2, 1, 1024, 1024, 32, True), ([9, 2, 3], [300, 5, 77], 4, 2, 64, 0, 16, False), ([3, 4], [2, 9], 3, 3, 10, 6, 16, False)])
def test_into_a_cache(dtype, past, new, heads, kv_heads, head_dim, rotated, page, heads_first):
    c = Paged(dtype, past, new, kv_heads, head_dim, page, heads_first=heads_first)
    g = torch.Generator(device=DEV).manual_seed(7)
    rows = c.tokens + 3  # (three more that belong to nobody)
    if c.offsets is None:
        rows = c.tokens
    qkv = torch.randn(rows, heads + 2 * kv_heads, head_dim, device=DEV, generator=g).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    qw, kw = torch.randn(heads, head_dim, device=DEV, generator=g).to(dtype), torch.randn(head_dim, device=DEV, generator=g).to(dtype)
    freqs = freqs_of(rotated) if rotated else None
    before_k, before_v = c.k.clone(), c.v.clone()
    q_out = torch.full_like(q, 7.0)
    eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, c.offsets, q=q, freqs=freqs, first_position=11, q_out=q_out, q_weight=qw,
                          k_weight=kw)
    assert (q_out[c.tokens:] == 7.0).all()
    written_k, written_v = before_k.clone(), before_v.clone()
    for i, (p, n) in enumerate(zip(past, new)):
        mine = slice(c.starts[i], c.starts[i] + n)
        positions = torch.arange(11 + p, 11 + p + n, device=DEV)
        check(q_out[mine], q[mine], qw, positions, freqs)
        got = c.read(c.k, c.table[i], p + n)[p:]
        check(got, k[mine], kw, positions, freqs)
        c.fill(written_k, c.table[i], p, got), c.fill(written_v, c.table[i], p, v[mine])
    # nothing else has changed
    for a, b in ((c.k, written_k), (c.v, written_v)):
        assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))


def test_keys_alone_and_one_of_the_norms():
    c, d = (Paged(torch.float16, [5, 9], [1, 1], 2, 64, 16) for _ in range(2))
    q, k, v = (torch.randn(2, n, 64, device=DEV).half() for n in (4, 2, 2))
    w, freqs, places = torch.randn(64, device=DEV).half(), freqs_of(64), c.lengths.long()
    assert eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, freqs=freqs, k_weight=w) is None
    want = eager.qk_norm_rotary(k, None, w, None, places, freqs)[0]
    for i, p in enumerate(c.past):
        assert torch.equal(c.read(c.k, c.table[i], p + 1)[p], want[i])
    # queries normalized, keys as without norms; no rotation
    got = eager.paged_kv_append(k, v, d.k, d.v, d.table, d.lengths, q=q, q_weight=w)
    assert torch.equal(got, eager.qk_norm_rotary(q, None, w, None, places)[0])
    for i, p in enumerate(d.past):
        assert torch.equal(d.read(d.k, d.table[i], p + 1)[p], k[i]) and torch.equal(d.read(d.v, d.table[i], p + 1)[p], v[i])


def test_pages_that_are_not_there():
    c = Paged(torch.float16, [5, 9], [1, 1], 2, 64, 16)
    c.table[1] = 999
    before = c.k.clone()
    q, k, v = (torch.randn(2, n, 64, device=DEV).half() for n in (4, 2, 2))
    w = torch.ones(64, device=DEV).half()
    got = eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, q=q, freqs=freqs_of(64), q_weight=w, k_weight=w)
    check(got, q, w, c.lengths.long(), freqs_of(64))
    c.fill(before, c.table[0], 5, c.read(c.k, c.table[0], 6)[5:])
    assert torch.equal(c.k.nan_to_num(5.0), before.nan_to_num(5.0))


def test_refusals():
    x, w, positions, freqs = torch.randn(3, 4, 64, device=DEV).half(), torch.ones(64, device=DEV).half(), torch.arange(3, device=DEV), freqs_of(64)
    for args, word in (((x, None, w, w, positions, freqs), "without k"), ((x, x[:2], w, w, positions, freqs), "fit"),
                       ((x, x, w[:32], w, positions, freqs), "q_weight"), ((x, x, w, w.float(), positions, freqs), "k_weight"),
                       ((x, x, w, w, positions[:2], freqs), "positions"), ((x, x, w, w, positions, freqs_of(128)), "freqs"),
                       ((x.cpu(), x, w, w, positions, freqs), "q")):
        with pytest.raises(ValueError, match=word):
            eager.qk_norm_rotary(*args)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="eps"):
            eager.qk_norm_rotary(x, x, w, w, positions, freqs, eps=eps)
    c = Paged(torch.float16, [5, 9, 1], [1, 1, 1], 4, 64, 16)
    with pytest.raises(ValueError, match="without q"):
        eager.paged_kv_append(x, x, c.k, c.v, c.table, c.lengths, freqs=freqs, q_weight=w)
    with pytest.raises(ValueError, match="k_weight"):
        eager.paged_kv_append(x, x, c.k, c.v, c.table, c.lengths, freqs=freqs, k_weight=w.view(1, 64))
