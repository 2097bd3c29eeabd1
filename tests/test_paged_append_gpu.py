"""Keys and values into a paged cache on the GPU, with the rotation on the way."""
import pytest
import torch

from aitemplate_amd import eager
from paged_common import DEV, Paged
from test_rotary_gpu import turned

pytestmark = pytest.mark.gpu


def allowed(want, size, dtype):
    return want.abs() * torch.finfo(dtype).eps / 2 * (1 + 1e-4) + size * 1e-6 + torch.finfo(dtype).smallest_normal


def check(c, k, v, q, freqs, interleaved, scale=1.0, first=0):
    """Appends and compares everything: queries, the new places, and that no other place changed."""
    before = c.k.clone(), c.v.clone()
    k0, v0, q0 = k.clone(), v.clone(), q.clone()
    got_q = eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, c.offsets, q=q, freqs=freqs, interleaved=interleaved,
                                  scale=scale, first_position=first)
    assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(q, q0)
    for i, (p, n) in enumerate(zip(c.past, c.new)):
        rows = slice(c.starts[i], c.starts[i + 1])
        places = torch.arange(p, p + n, device=DEV)
        if freqs is None:
            want_k, want_q = k[rows], q[rows]
            assert torch.equal(got_q[rows], want_q)
        else:
            want_q, size = turned(q[rows], places + first, freqs, interleaved, scale)
            assert ((got_q[rows].double() - want_q).abs() <= allowed(want_q, size, c.dtype)).all()
            want_k, size = turned(k[rows], places + first, freqs, interleaved, scale)
        keep = places >= 0
        places = places[keep]
        pages, slots = c.table[i][places // c.page].long(), places % c.page
        if freqs is None:
            assert torch.equal(c.k[pages, slots], want_k[keep])
        else:
            assert ((c.k[pages, slots].double() - want_k[keep]).abs() <= allowed(want_k, size, c.dtype)[keep]).all()
        assert torch.equal(c.v[pages, slots], v[rows][keep])
        for now, was in zip((c.k, c.v), before):
            was[pages, slots] = now[pages, slots]
    for now, was in zip((c.k, c.v), before):
        assert torch.equal(now.nan_to_num(7.0), was.nan_to_num(7.0))


def operands(c, heads, kv_heads, head_dim):
    qkv = torch.randn(c.tokens, heads + 2 * kv_heads, head_dim, device=DEV).to(c.dtype)
    return qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], qkv[:, :heads]


SIZES = [
    # past, new, heads, kv_heads, head_dim, rotated, page
    ([0], [1], 1, 1, 64, 64, 16),
    ([15, 16, 17, 0, 4095], [1, 1, 1, 1, 1], 8, 2, 128, 128, 16),
    (list(range(70)), [1] * 70, 4, 4, 64, 32, 32),
    ([3, 0, 40], [5, 17, 1], 6, 3, 80, 40, 16),
    ([0, 5, 7, 31], [0, 130, 0, 33], 7, 1, 96, 96, 64),
    ([10, 2], [300, 257], 32, 8, 128, 64, 256),
    ([4, 9], [3, 6], 2, 2, 10, 6, 1),
    ([4, 9], [3, 6], 3, 1, 65, 0, 7),
    ([i % 9 for i in range(200)], [(3 * i) % 7 for i in range(200)], 2, 1, 64, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("past,new,heads,kv_heads,head_dim,rotated,page", SIZES)
def test_append(dtype, heads_first, interleaved, past, new, heads, kv_heads, head_dim, rotated, page):
    c = Paged(dtype, past, new, kv_heads, head_dim, page, heads_first=heads_first)
    freqs = eager.rotary_frequencies(rotated, device=DEV)[0] if rotated else None
    check(c, *operands(c, heads, kv_heads, head_dim), freqs, interleaved)


def test_scale_and_first_position():
    c = Paged(torch.float16, [5, 6], [2, 3], 2, 64, 16)
    freqs, scale = eager.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=2048, device=DEV)
    check(c, *operands(c, 4, 2, 64), freqs, False, scale, 100000)


def test_rows_of_nobody_and_places_without_a_page():
    dtype, heads, kv_heads, D = torch.bfloat16, 4, 2, 64
    c = Paged(dtype, [14, 3, 0], [5, 2, 4], kv_heads, D, 16)
    # rows behind the last sequence; a sequence whose second page is missing; one whose pages lie outside the cache
    rows = c.tokens + 6
    qkv = torch.randn(rows, heads + 2 * kv_heads, D, device=DEV).to(dtype)
    c.table[0, 1] = -7
    c.table[2, 0] = c.k.shape[0]
    before = c.k.clone(), c.v.clone()
    out = torch.full((rows, heads, D), 5.0, device=DEV, dtype=dtype)
    freqs = eager.rotary_frequencies(D, device=DEV)[0]
    k, v, q = qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], qkv[:, :heads]
    got = eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, c.offsets, q=q, freqs=freqs, q_out=out)
    assert got is out and (out[c.tokens:] == 5.0).all() and torch.isfinite(out).all()
    want, size = turned(q[:5], torch.arange(14, 19, device=DEV), freqs, False)
    assert ((out[:5].double() - want).abs() <= allowed(want, size, dtype)).all()
    page = c.table[0, 0].long()
    assert torch.equal(c.v[page, 14:16], v[:2])
    own = c.table[1, 0].long()
    assert torch.equal(c.v[own, 3:5], v[5:7])
    for now, was in zip((c.k, c.v), before):
        was[page, 14:16], was[own, 3:5] = now[page, 14:16], now[own, 3:5]
        assert torch.equal(now.nan_to_num(7.0), was.nan_to_num(7.0))
    # lengths below zero (a sequence that is not there) and beyond the table: nothing is written
    k_now, v_now = c.k.clone(), c.v.clone()
    lengths = torch.tensor([-100, 1 << 30, 32], dtype=torch.int32, device=DEV)
    eager.paged_kv_append(k, v, c.k, c.v, c.table, lengths, c.offsets, q=q, freqs=freqs)
    assert torch.equal(c.k.nan_to_num(7.0), k_now.nan_to_num(7.0)) and torch.equal(c.v.nan_to_num(7.0), v_now.nan_to_num(7.0))


def test_without_queries_and_in_place():
    c = Paged(torch.float16, [1, 2], [1, 1], 2, 64, 16)
    k, v, q = operands(c, 4, 2, 64)
    freqs = eager.rotary_frequencies(64, device=DEV)[0]
    assert eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths) is None
    assert torch.equal(c.k[c.table[0, 0].long(), 1], k[0])
    assert eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, q=q) is q
    want = eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, q=q, freqs=freqs)
    assert eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, q=q, freqs=freqs, q_out=q) is q
    assert torch.equal(q, want)


def test_offsets_past_32_bits():
    # places of a cache beyond 2^32 elements, reached through the page stride of a view (5 GiB each)
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GiB of free memory")
    pages, D = 5, 64
    k_all, v_all = (torch.empty(5 * (1 << 30) // 2 + 16 * D, dtype=torch.float16, device=DEV) for _ in range(2))
    stride = (1 << 29)
    k_cache, v_cache = (t.as_strided((pages, 16, 1, D), (stride, D, D, 1)) for t in (k_all, v_all))
    k, v = (torch.randn(1, 1, D, device=DEV).half() for _ in range(2))
    table = torch.tensor([[4]], dtype=torch.int32, device=DEV)
    eager.paged_kv_append(k, v, k_cache, v_cache, table, torch.tensor([15], dtype=torch.int32, device=DEV))
    at = 4 * stride + 15 * D
    assert torch.equal(k_all[at:at + D], k[0, 0]) and torch.equal(v_all[at:at + D], v[0, 0])


def test_more_tokens_than_one_launch_takes():
    # (2^24 workgroups of 64 tokens and two more)
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of free memory")
    tokens, page = (1 << 30) + 70, 1 << 20
    k = torch.ones(tokens, 1, 2, dtype=torch.float16, device=DEV)
    k_cache, v_cache = (torch.zeros(tokens // page + 1, page, 1, 2, dtype=torch.float16, device=DEV) for _ in range(2))
    table = torch.arange(k_cache.shape[0], dtype=torch.int32, device=DEV)[None]
    lengths, offsets = (torch.tensor(at, dtype=torch.int32, device=DEV) for at in ([0], [0, tokens]))
    eager.paged_kv_append(k, k, k_cache, v_cache, table, lengths, offsets)
    for cache in (k_cache, v_cache):
        assert (cache.view(-1)[:2 * tokens] == 1).all() and not cache.view(-1)[2 * tokens:].any()


def test_captured_and_replayed_while_lengths_grow():
    c = Paged(torch.float16, [3, 14], [1, 1], 2, 64, 16, spare=8)
    c.table = torch.cat((c.table, c.spare[:4].int().view(2, 2)), 1).contiguous()
    freqs = eager.rotary_frequencies(64, device=DEV)[0]
    k, v, q = operands(c, 4, 2, 64)
    lengths, out = c.lengths.clone(), torch.empty(2, 4, 64, dtype=torch.float16, device=DEV)
    eager.paged_kv_append(k, v, c.k, c.v, c.table, lengths, q=q, freqs=freqs, q_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eager.paged_kv_append(k, v, c.k, c.v, c.table, lengths, q=q, freqs=freqs, q_out=out)
    for _ in range(5):
        k.normal_(), v.normal_(), q.normal_()
        lengths += 1
        graph.replay()
        torch.cuda.synchronize()
        got = c.k.clone(), c.v.clone(), out.clone()
        want = eager.paged_kv_append(k, v, c.k, c.v, c.table, lengths, q=q, freqs=freqs)
        assert torch.equal(got[2], want)
        assert torch.equal(got[0].nan_to_num(7.0), c.k.nan_to_num(7.0)) and torch.equal(got[1].nan_to_num(7.0), c.v.nan_to_num(7.0))
