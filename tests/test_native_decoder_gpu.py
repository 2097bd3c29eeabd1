"""The decoder operators' calls through the extension module and through the Python path: the same results, and arguments that
the module leaves to the Python path are served or refused there."""
import pytest
import torch

from aitemplate_amd import _kernels, eager
from paged_common import DEV, Paged

pytestmark = pytest.mark.gpu


def calls():
    g = torch.Generator(device=DEV).manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).half()

    x = normal(6, 4, 64)
    freqs, scale = eager.rotary_frequencies(64, device=DEV)
    a, a_scale = eager.quantize_rows(normal(6, 128))
    b, b_scale = eager.quantize_rows(normal(24, 128))
    c = Paged(torch.float16, [20, 3, 40], [1, 3, 2], 2, 64, 16, 33)
    q, k, v = normal(6, 8, 64), normal(6, 2, 64), normal(6, 2, 64)
    cache = (c.k, c.v, c.table, c.lengths, c.offsets)
    positions = torch.arange(6, device=DEV)
    shared = dict(prefix_table=c.prefix_table, prefix_length=33)
    eager.paged_kv_append(k, v, *cache)
    return {
        "quantize": lambda: eager.quantize_rows(x),
        "quantize_pitch": lambda: eager.quantize_rows(x.view(6, 256)[:, :100]),
        "int8": lambda: eager.gemm_rcr_int8(a, b, a_scale, b_scale, dtype=torch.bfloat16),
        "int8_bias": lambda: eager.gemm_rcr_int8(a.view(2, 3, 128), b, a_scale.view(2, 3), b_scale, normal(24) * 0),
        "rotary": lambda: eager.rotary_embedding(x, positions, freqs),
        "rotary_batch": lambda: eager.rotary_embedding(x.view(2, 3, 4, 64), positions[:3].int(), freqs, True, 0.5, True),
        "rotary_batches": lambda: eager.rotary_embedding(x.view(2, 3, 4, 64), positions.view(2, 3), freqs, inverse=True),
        "rotary_out": lambda: eager.rotary_embedding(x, positions, freqs, out=torch.empty(4, 6, 64, device=DEV).half().transpose(0, 1)),
        "append": lambda: (eager.paged_kv_append(k, v, *cache, q=q, freqs=freqs), c.k.nan_to_num(0), c.v.nan_to_num(0)),
        "append_scaled": lambda: (eager.paged_kv_append(k, v, *cache, q=q, freqs=freqs, interleaved=True, scale=1.5, first_position=7,
                                                        q_out=torch.empty_like(q)), c.k.nan_to_num(0)),
        "append_as_it_is": lambda: (eager.paged_kv_append(k, v, *cache, q=q), c.k.nan_to_num(0)),
        "append_keys": lambda: (eager.paged_kv_append(k, v, *cache, freqs=freqs), c.k.nan_to_num(0), c.v.nan_to_num(0)),
        "append_bare": lambda: (eager.paged_kv_append(k, v, *cache), c.k.nan_to_num(0), c.v.nan_to_num(0)),
        "attention": lambda: eager.prefix_attention(q, *cache),
        "attention_shared": lambda: eager.prefix_attention(q, *cache, **shared),
        "attention_scaled": lambda: eager.prefix_attention(q, *cache, scale=0.2, out=torch.empty_like(q), **shared),
    }


@pytest.mark.parametrize("name", list(calls()) if torch.cuda.is_available() else [])
def test_both_paths(name, monkeypatch):
    assert not isinstance(eager._native_decoder, _kernels._NoNative)
    call = calls()[name]
    leaves = lambda r: r if isinstance(r, tuple) else (r,)  # noqa: E731
    native = [t if t is None else t.clone() for t in leaves(call())]

    class Counted:  # the module takes each of these calls
        taken = 0

        def __getattr__(self, f):
            def run(*args):
                r = getattr(_kernels.load_native("_native_decoder"), f)(*args)
                Counted.taken += r is not NotImplemented
                return r
            return run

    monkeypatch.setattr(eager, "_native_decoder", Counted())
    call()
    assert Counted.taken >= 1
    monkeypatch.setattr(eager, "_native_decoder", _kernels._NoNative())
    for a, b in zip(native, leaves(call())):
        assert (a is None and b is None) or (a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b))


@pytest.mark.parametrize("python_only", [False, True])
def test_refused_either_way(python_only, monkeypatch):
    if python_only:
        monkeypatch.setattr(eager, "_native_decoder", _kernels._NoNative())
    x = torch.randn(6, 4, 64, device=DEV).half()
    freqs, positions = torch.ones(32, device=DEV), torch.arange(6, device=DEV)
    i8, s = torch.zeros(6, 64, dtype=torch.int8, device=DEV), torch.ones(6, device=DEV)
    c = Paged(torch.float16, [20, 3], [1, 1], 2, 64, 16, 33)
    cache = (c.k, c.v, c.table, c.lengths)
    q, k = torch.randn(2, 8, 64, device=DEV).half(), torch.randn(2, 2, 64, device=DEV).half()
    refused = [
        lambda: eager.quantize_rows(x.float()),
        lambda: eager.quantize_rows(x.transpose(0, 1)),
        lambda: eager.quantize_rows(x[0], out=torch.empty(4, 63, dtype=torch.int8, device=DEV)),
        lambda: eager.gemm_rcr_int8(i8, i8, s, s, dtype=torch.float32),
        lambda: eager.gemm_rcr_int8(i8, i8[:, :32], s, s),
        lambda: eager.gemm_rcr_int8(i8, i8, s[:5], s),
        lambda: eager.gemm_rcr_int8(i8, i8, s, s.half()),
        lambda: eager.gemm_rcr_int8(i8, i8, s, s, bias=s),
        lambda: eager.gemm_rcr_int8(i8.half(), i8, s, s),
        lambda: eager.rotary_embedding(x, positions[:5], freqs),
        lambda: eager.rotary_embedding(x, positions.float(), freqs),
        lambda: eager.rotary_embedding(x, positions, torch.ones(33, device=DEV)),
        lambda: eager.rotary_embedding(x, positions, freqs.half()),
        lambda: eager.rotary_embedding(x, positions, freqs, out=x[:5]),
        lambda: eager.rotary_embedding(x.transpose(1, 2), positions, freqs[:2]),
        lambda: eager.rotary_embedding(x.float(), positions, freqs),
        lambda: eager.paged_kv_append(k, k[:1], *cache),
        lambda: eager.paged_kv_append(k, k, c.k, c.v[:-1], c.table, c.lengths),
        lambda: eager.paged_kv_append(k[:, :1], k[:, :1], *cache),
        lambda: eager.paged_kv_append(k.bfloat16(), k, *cache),
        lambda: eager.paged_kv_append(k, k, *cache, q=q[:1]),
        lambda: eager.paged_kv_append(k, k, *cache, q_out=q),
        lambda: eager.paged_kv_append(k, k, c.k, c.v, c.table.long(), c.lengths),
        lambda: eager.paged_kv_append(k, k, c.k, c.v, c.table[:1], c.lengths),
        lambda: eager.paged_kv_append(k[:1], k[:1], *cache),
        lambda: eager.paged_kv_append(k, k, *cache, offsets=c.lengths),
        lambda: eager.prefix_attention(q[0], *cache),
        lambda: eager.prefix_attention(q, c.k, c.v, c.table.t(), c.lengths),
        lambda: eager.prefix_attention(q, *cache, prefix_length=5),
        lambda: eager.prefix_attention(q, *cache, prefix_table=c.prefix_table.long(), prefix_length=5),
        lambda: eager.prefix_attention(q, *cache, out=q[:1]),
        lambda: eager.prefix_attention(q.float(), *cache),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    late = [  # refused by the library
        lambda: eager.prefix_attention(q, *cache, prefix_table=c.prefix_table, prefix_length=49),
        lambda: eager.prefix_attention(q[:, :7], *cache),
        lambda: eager.prefix_attention(q, c.k[:, :8], c.v[:, :8], c.table, c.lengths),
        lambda: eager.prefix_attention(q[:, :, :60], c.k[..., :60], c.v[..., :60], c.table, c.lengths),
        lambda: eager.gemm_rcr_int8(i8, i8, s, s, algo=10 ** 6),
    ]
    for i, call in enumerate(late):
        with pytest.raises(RuntimeError):
            call()
            print("not refused:", i)
    torch.cuda.synchronize()
