"""Adapters beside a projection, normalized heads and log probabilities without a GPU: as graph ops (shapes, generated calls,
refusals), and what the C ABI and the eager calls refuse.  Nothing here launches anything."""
import ctypes

import pytest
import torch

from aitemplate_amd import _kernels, eager
from aitemplate_amd.compiler import ops
from aitemplate_amd.frontend import IntImm, IntVar
from test_decoder_ops_cpu import cache as graph_cache
from test_decoder_ops_cpu import generated, tensor
from test_decoder_refusals_cpu import P, cache, refused


def lora(dtype=0, algo=-1, x=P, w=P, bias=None, a=P, b=P, adapters=P, scales=P, y=P, M=2, N=8, K=64, rank=16, n=3, ldx=64, ldw=64, ldy=8,
         workspace=P, nbytes=1 << 20):
    return _kernels.load().aitamd_gemm_rcr_lora(dtype, algo, x, w, bias, a, b, adapters, scales, y, M, N, K, rank, n, ldx, ldw, ldy, workspace,
                                                nbytes, None)


def test_gemm_rcr_lora_refusals():
    lib = _kernels.load()
    refused(lora(dtype=2), "dtype")
    refused(lora(M=-1), "negative")
    refused(lora(n=-1), "negative")
    refused(lora(rank=0), "rank")
    refused(lora(rank=1025), "rank")
    refused(lora(N=1 << 31, ldy=1 << 31), "large")
    refused(lora(x=None), "null")
    refused(lora(b=None), "null")
    refused(lora(adapters=None), "null")
    refused(lora(y=None), "null")
    refused(lora(ldx=63), "pitch")
    refused(lora(ldy=7), "pitch")
    refused(lora(adapters=ctypes.c_void_p(66)), "aligned")
    refused(lora(scales=ctypes.c_void_p(65)), "aligned")
    refused(lora(workspace=None), "workspace")
    refused(lora(nbytes=4096 + 2 * 64 - 1), "workspace")
    refused(lora(workspace=ctypes.c_void_p(72)), "workspace", "aligned")
    assert lora(M=0, x=None, y=None, workspace=None) == 0
    # the tables of products with adapters take them: not through the other entry points
    assert lib.aitamd_gemm_num_algos(0, 4) > 0 and lib.aitamd_gemm_num_algos(1, 5) > 0 and lib.aitamd_gemm_num_algos(3, 4) == 0
    refused(lib.aitamd_gemm_rcr(0, 4, -1, P, P, None, None, None, P, 2, 8, 64, 64, 64, 8, 8, None), "dtype")
    assert all(name.startswith("gemm_rcr_bf16_lora_") for name in _kernels.gemm_algo_names(1, 5))


def test_workspaces():
    lib = _kernels.load()
    # the counters of tiles that are shared, then 16 bytes for a row's rank in two parts
    assert lib.aitamd_gemm_lora_workspace_bytes(0, 0, 0, 5, 64, 64, 9) == 4096 + 5 * 64
    assert lib.aitamd_gemm_lora_workspace_bytes(0, -1, 0, 64, 6144, 4096, 16) > 4096 + 64 * 64
    for bad in ((2, -1, 0, 5, 64, 64, 9), (0, -1, 0, 0, 64, 64, 9), (0, -1, 0, 5, 64, 64, 0), (0, -1, 0, 5, 64, 64, 1025)):
        assert lib.aitamd_gemm_lora_workspace_bytes(*bad) == 0
    assert lib.aitamd_token_logprobs_workspace_bytes(4096, 32000, 20) == 0
    assert lib.aitamd_token_logprobs_workspace_bytes(1, 131072, 20) == 16 * (16 + 160)
    assert lib.aitamd_token_logprobs_workspace_bytes(1, 131072, 65) == 0


def norm(dtype=0, q=True, k=True, x=P, out=P, weight=P, heads=4, positions=P, freqs=P, batch=1, seq=2, head_dim=64, rotated=64, eps=1e-6):
    h = _kernels.Heads(x, out, heads, 0, 256, 64, 0, 256, 64, weight, 0)
    return _kernels.load().aitamd_qk_norm_rotary(dtype, h if q else None, h if k else None, positions, 0, freqs, batch, seq, head_dim, rotated, 0, 1,
                                                 eps, 1.0, 0, None)


def test_qk_norm_rotary_refusals():
    refused(norm(dtype=2), "dtype")
    refused(norm(seq=-1), "negative")
    refused(norm(heads=-1), "negative")
    refused(norm(head_dim=1026, rotated=0), "head_dim")
    refused(norm(rotated=63), "rotated")
    refused(norm(rotated=66), "rotated")
    refused(norm(x=None), "null")
    refused(norm(out=None, q=False), "null")
    refused(norm(positions=None), "null")
    refused(norm(freqs=None), "freqs")
    refused(norm(batch=1 << 20, seq=1 << 20), "large")
    refused(norm(heads=1 << 30), "large")
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(norm(eps=eps), "eps")
    assert norm(seq=0, x=None, out=None) == 0 and norm(q=False, k=False) == 0


def append(c=None, dtype=0, k=P, v=P, q=P, q_out=P, heads=4, q_weight=P, k_weight=P, eps=1e-6, freqs=P, rotated=64):
    return _kernels.load().aitamd_paged_kv_append_norm(dtype, c, k, 128, 64, v, 128, 64, q, 256, 64, q_out, 256, 64, heads, q_weight, 0, k_weight, 0,
                                                       eps, freqs, rotated, 0, 1.0, 0, None)


def test_paged_kv_append_norm_refusals():
    for weights in (dict(), dict(q_weight=None), dict(q_weight=None, k_weight=None)):
        refused(append(None, **weights), "null", "cache")
        refused(append(cache(), dtype=7, **weights), "dtype")
        refused(append(cache(page_size=0), **weights), "page_size")
        refused(append(cache(tokens=4), **weights), "without offsets")
        refused(append(cache(lengths=None), **weights), "null")
        refused(append(cache(table=66), **weights), "aligned")
        refused(append(cache(), k=None, **weights), "null")
        refused(append(cache(), q_out=None, **weights), "q_out")
        refused(append(cache(), freqs=None, **weights), "freqs")
        refused(append(cache(), rotated=65, **weights), "rotated")
        refused(append(cache(), heads=1 << 30, **weights), "large")
        assert append(cache(tokens=0, batch=0), **weights) == 0
    refused(append(cache(), eps=-1.0), "eps")


def logprobs(dtype=0, logits=P, tokens=P, wide=1, logprob=P, entropy=P, rank=P, top_logprob=P, top_token=P, rows=2000, V=1000, ld=1000, top=0, scale=1.0,
             workspace=None, nbytes=0):
    return _kernels.load().aitamd_token_logprobs(dtype, logits, tokens, wide, logprob, entropy, rank, top_logprob, top_token, rows, V, ld, top, scale,
                                                 workspace, nbytes, None)


def test_token_logprobs_refusals():
    refused(logprobs(dtype=2), "dtype")
    refused(logprobs(rows=-1), "negative")
    refused(logprobs(top=65), "top")
    refused(logprobs(top=-1), "top")
    refused(logprobs(V=10, top=11), "top")
    refused(logprobs(V=0), "no tokens")
    refused(logprobs(rows=1 << 31), "large")
    refused(logprobs(V=1 << 31, ld=1 << 31), "large")
    refused(logprobs(ld=999), "pitch")
    for name in ("logits", "tokens", "logprob", "entropy", "rank"):
        refused(logprobs(**{name: None}), "null")
    refused(logprobs(top=3, top_token=None), "null")
    refused(logprobs(logits=ctypes.c_void_p(65)), "aligned")
    refused(logprobs(dtype=8, logits=ctypes.c_void_p(66)), "aligned")
    refused(logprobs(tokens=ctypes.c_void_p(68)), "aligned")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(logprobs(scale=scale), "scale")
    refused(logprobs(rows=1, V=100000, ld=100000), "workspace")
    refused(logprobs(rows=1, V=100000, ld=100000, workspace=ctypes.c_void_p(72), nbytes=1 << 20), "workspace", "aligned")
    assert logprobs(rows=0, logits=None) == 0


def test_ranges_ends():
    """A scale whose product with log2(e) is beyond 32 bits; ranks from 1025 on."""
    refused(logprobs(scale=3e38), "scale")
    with pytest.raises(RuntimeError):
        ops.token_logprobs(scale=3e38)
    m, n = IntVar(values=[1, 64], name="m"), IntVar(values=[1, 9], name="n")
    x, w, of = tensor("x", [m, 256]), tensor("w", [96, 256]), tensor("of", [m], "int32")
    ops.gemm_rcr_lora()(x, w, tensor("a", [n, 1024, 256]), tensor("b", [n, 96, 1024]), of)
    with pytest.raises(RuntimeError):
        ops.gemm_rcr_lora()(x, w, tensor("a", [n, 1025, 256]), tensor("b", [n, 96, 1025]), of)


def test_eager_calls_take_gpu_tensors_only():
    x = torch.zeros(2, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        eager.gemm_rcr_lora(x, x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        eager.qk_norm_rotary(x, x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        eager.paged_kv_append(x, x, x, x, x, x, k_weight=x)
    with pytest.raises(ValueError, match="GPU"):
        eager.token_logprobs(x, x)


def test_lora_op():
    m, n = IntVar(values=[1, 64], name="m"), IntVar(values=[1, 9], name="n")
    x, w, a, b = tensor("x", [m, 256]), tensor("w", [96, 256]), tensor("a", [n, 8, 256]), tensor("b", [n, 96, 8])
    of, scales, bias = tensor("of", [m], "int32"), tensor("scales", [n], "float32"), tensor("bias", [96])
    op = ops.gemm_rcr_lora()
    y = op(x, w, a, b, of, scales, bias)
    assert y._attrs["shape"] == [m, IntImm(96)] and y._attrs["dtype"] == "float16" and op._attrs["workspace"] >= 4096 + 64 * 32
    source, decl, call = generated(op, "project")
    assert "aitamd_gemm_rcr_lora(0, -1" in source and "aitamd_gemm_table_1_4" in source and decl.endswith(";") and "project(" in call
    op = ops.gemm_rcr_lora()
    op(x, w, a, b, of)
    source, _, call = generated(op, "plain")
    assert "aitamd_gemm_table_0_4" in source and "of, nullptr, nullptr," in call
    for bad in ((x, w, a, b, tensor("o", [m])), (x, w, a, b, tensor("o", [n], "int32")), (x, w, tensor("a", [n, 8, 128]), b, of),
                (x, w, a, tensor("b", [n, 96, 16]), of), (x, tensor("w", [96, 256], "bfloat16"), a, b, of), (x, w, a, b, of, tensor("s", [n])),
                (x, w, a, b, of, scales, tensor("t", [95])), (x, w, a, b, of, tensor("s", [3], "float32"))):
        with pytest.raises(RuntimeError):
            ops.gemm_rcr_lora()(*bad)


def test_norm_op():
    s = IntVar(values=[1, 64], name="s")
    q, k, positions, freqs = tensor("q", [2, s, 4, 64]), tensor("k", [2, s, 2, 64]), tensor("p", [s], "int32"), tensor("f", [16], "float32")
    qw, kw = tensor("qw", [64]), tensor("kw", [2, 64])
    op = ops.qk_norm_rotary(eps=1e-5, interleaved=True)
    a, b = op(q, k, qw, kw, positions, freqs)
    assert a._attrs["shape"] == q._attrs["shape"] and b._attrs["shape"] == k._attrs["shape"]
    source, _, call = generated(op, "heads")
    assert "aitamd_qk_norm_rotary(0, &q_heads, &k_heads" in source and "k_weight, 64}" in source and "q_weight, 0}" in source and "heads(" in call
    for bad in ((q, tensor("k", [2, s, 2, 32]), qw, kw, positions, freqs), (q, k, tensor("w", [32]), kw, positions, freqs),
                (q, k, qw, tensor("w", [4, 64]), positions, freqs), (q, k, qw, kw, tensor("p", [3], "int32"), freqs),
                (q, k, qw, kw, positions, tensor("f", [33], "float32")), (q, tensor("k", [2, s, 2, 64], "bfloat16"), qw, kw, positions, freqs)):
        with pytest.raises(RuntimeError):
            ops.qk_norm_rotary()(*bad)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rotary(eps=-1.0)


def test_append_op_with_norms():
    b = IntVar(values=[1, 8], name="b")
    q, k, v = tensor("q", [b, 8, 64]), tensor("k", [b, 2, 64]), tensor("v", [b, 2, 64])
    table, lengths, freqs = tensor("table", [b, 3], "int32"), tensor("lengths", [b], "int32"), tensor("f", [32], "float32")
    w, each = tensor("norm", [64]), tensor("norms", [8, 64])
    op = ops.paged_kv_append(eps=1e-5)
    op(q, k, v, *graph_cache(), table, lengths, freqs, q_weight=each, k_weight=w)
    source, _, call = generated(op, "put")
    assert "aitamd_paged_kv_append_norm(0, &cache" in source and "q_weight, 64, k_weight, 0, " in source and "norms, norm, stream" in call
    op = ops.paged_kv_append()
    op(q, k, v, *graph_cache(), table, lengths, freqs, k_weight=w)
    assert "nullptr, norm, stream" in generated(op, "put")[2]
    with pytest.raises(RuntimeError):
        ops.paged_kv_append()(q, k, v, *graph_cache(), table, lengths, freqs, k_weight=each)


def test_logprobs_op():
    m = IntVar(values=[1, 64], name="m")
    logits, tokens = tensor("logits", [m, 1000], "float32"), tensor("tokens", [m], "int64")
    op = ops.token_logprobs(top=5, scale=0.5)
    outs = op(logits, tokens)
    assert [t._attrs["dtype"] for t in outs] == ["float32", "float32", "int32", "float32", "int32"]
    assert outs[0]._attrs["shape"] == [m] and outs[4]._attrs["shape"] == [m, IntImm(5)]
    source, _, call = generated(op, "score")
    assert "aitamd_token_logprobs(8, logits, tokens, 1," in source and "5, 0.5f, workspace + 4096" in source and "score(" in call
    op = ops.token_logprobs()
    assert len(op(tensor("logits", [2, 1000]), tensor("tokens", [2], "int32"))) == 3
    assert "nullptr, nullptr, logits" in generated(op, "score")[2]
    for bad in ((tensor("l", [m, 1000], "int32"), tokens), (logits, tensor("t", [m], "float32")), (logits, tensor("t", [3], "int32")),
                (tensor("l", [m, 4]), tokens), (tensor("l", [1000]), tokens)):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(top=5)(*bad)
    for kw in (dict(top=65), dict(top=-1), dict(scale=0.0)):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(**kw)
