"""Calls that the decoder operators refuse, at the C ABI and in the eager calls; nothing here launches anything."""
import ctypes
import math

import pytest
import torch

from aitemplate_amd import _kernels, eager

P = ctypes.c_void_p(64)  # never followed: every call below is refused or has nothing to do


def refused(rc, *words):
    message = _kernels.last_error()
    assert rc != 0 and all(w in message for w in words), (rc, message)


def quantize(dtype=0, x=P, q=P, scale=P, rows=2, columns=64, ldx=64, ldq=64):
    return _kernels.load().aitamd_quantize_rows(dtype, x, q, scale, rows, columns, ldx, ldq, None)


def test_quantize_rows():
    refused(quantize(dtype=2), "dtype")
    refused(quantize(rows=-1), "negative")
    refused(quantize(x=None), "null")
    refused(quantize(scale=None), "null")
    refused(quantize(ldx=63), "pitch")
    refused(quantize(columns=1 << 31, ldx=1 << 31, ldq=1 << 31), "large")
    assert quantize(rows=0, x=None, q=None, scale=None) == 0


def int8(dtype=0, algo=-1, a=P, b=P, scale_a=P, scale_b=P, bias=None, c=P, M=2, N=8, K=64, lda=64, ldb=64, ldc=8):
    return _kernels.load().aitamd_gemm_rcr_int8(dtype, algo, a, b, scale_a, scale_b, bias, c, M, N, K, lda, ldb, ldc, None, 0, None)


def test_gemm_rcr_int8():
    lib = _kernels.load()
    refused(int8(dtype=2), "dtype")
    refused(int8(M=-1), "negative")
    refused(int8(M=1 << 31), "large")
    refused(int8(K=131072, lda=131072, ldb=131072), "131071")
    refused(int8(a=None), "null")
    refused(int8(scale_b=None), "null")
    refused(int8(c=None), "null")
    refused(int8(lda=63), "pitch")
    refused(int8(ldc=7), "pitch")
    refused(int8(scale_a=ctypes.c_void_p(66)), "aligned")
    refused(int8(algo=0, K=63), "dwords")
    refused(int8(algo=999), "range")
    assert int8(M=0, a=None, c=None) == 0
    # the tables of 8-bit integers take scales: not through the other entry points
    assert lib.aitamd_gemm_num_algos(0, 2) > 0 and lib.aitamd_gemm_num_algos(3, 2) == 0
    refused(lib.aitamd_gemm_rcr(0, 2, -1, P, P, None, None, None, P, 2, 8, 64, 64, 64, 8, 8, None), "dtype")
    for name in _kernels.gemm_algo_names(1, 3):
        assert name.startswith("gemm_rcr_i8_bf16_")


def rotary(dtype=0, x=P, out=P, positions=P, freqs=P, batch=1, seq=2, heads=2, head_dim=64, rotated=64):
    return _kernels.load().aitamd_rotary_embedding(dtype, x, out, positions, 0, freqs, batch, seq, heads, head_dim, rotated, 0, 128, 64, 0,
                                                   128, 64, 0, 1, 1.0, 0, 0, None)


def test_rotary_embedding():
    refused(rotary(dtype=-1), "dtype")
    refused(rotary(seq=-1), "negative")
    refused(rotary(rotated=63), "rotated")
    refused(rotary(rotated=66), "rotated")
    refused(rotary(head_dim=1026, rotated=0), "head_dim")
    refused(rotary(x=None), "null")
    refused(rotary(freqs=None), "freqs")
    refused(rotary(batch=1 << 20, seq=1 << 20), "large")
    refused(rotary(heads=1 << 30), "large")
    assert rotary(seq=0, x=None, out=None, positions=None) == 0


def cache(**changed):
    c = _kernels.PagedCache(64, 64, 8, 16, 2, 64, 2048, 128, 64, 2048, 128, 64, 64, 4, 4, 64, None, 3, 3)
    for name, value in changed.items():
        setattr(c, name, value)
    return c


def append(c=None, dtype=0, k=P, v=P, q=P, q_out=P, heads=4, freqs=P, rotated=64):
    return _kernels.load().aitamd_paged_kv_append(dtype, c, k, 128, 64, v, 128, 64, q, 256, 64, q_out, 256, 64, heads, freqs, rotated, 0,
                                                  1.0, 0, None)


def test_paged_kv_append():
    refused(append(None), "null", "cache")
    refused(append(cache(), dtype=7), "dtype")
    refused(append(cache(page_size=0)), "page_size")
    refused(append(cache(batch=-1)), "negative")
    refused(append(cache(tokens=4)), "without offsets")
    refused(append(cache(lengths=None)), "null")
    refused(append(cache(table=None)), "null")
    refused(append(cache(k=None)), "null")
    refused(append(cache(max_pages=1 << 28)), "large")
    refused(append(cache(table=66)), "aligned")
    refused(append(cache(lengths=65)), "aligned")
    refused(append(cache(), k=None), "null")
    refused(append(cache(), q_out=None), "q_out")
    refused(append(cache(), freqs=None), "freqs")
    refused(append(cache(), rotated=65), "rotated")
    refused(append(cache(), heads=1 << 30), "large")
    assert append(cache(tokens=0, batch=0)) == 0


def attention(c=None, dtype=0, q=P, out=P, heads=4, table=P, pages=4, length=0, workspace=None, nbytes=0,
              scale=0.125):
    return _kernels.load().aitamd_prefix_attention(dtype, c, q, 256, 64, out, 256, 64, heads, table, pages, length, scale, workspace,
                                                   nbytes, None)


def workspace_bytes(c, heads=4, length=0):
    return _kernels.load().aitamd_prefix_attention_workspace_bytes(c, heads, length)


def test_prefix_attention():
    refused(attention(None), "null", "cache")
    refused(attention(cache(), dtype=2), "dtype")
    refused(attention(cache(page_size=24)), "page_size", "16")
    refused(attention(cache(head_dim=60)), "head_dim")
    refused(attention(cache(head_dim=264)), "head_dim")
    refused(attention(cache(), heads=5), "multiple")
    refused(attention(cache(kv_heads=0)), "multiple")
    refused(attention(cache(), q=None), "null")
    refused(attention(cache(v=None)), "null")
    refused(attention(cache(), length=5, table=None), "null")
    refused(attention(cache(), length=65), "prefix", "pages")
    refused(attention(cache(), length=-1), "negative")
    refused(attention(cache(k=72)), "aligned")
    refused(attention(cache(), table=ctypes.c_void_p(66), length=5), "aligned")
    refused(attention(cache(k_page_stride=-8)), "stride")
    refused(attention(cache(page_size=1 << 20, max_pages=1, v_slot_stride=1 << 12)), "large")
    refused(attention(cache(v_head_stride=65)), "strides")
    refused(attention(cache(k_slot_stride=56)), "stride")
    refused(attention(cache(k_slot_stride=1 << 25)), "stride")
    refused(attention(cache(tokens=2)), "without offsets")
    refused(attention(cache(max_pages=1 << 27)), "large")
    refused(attention(cache(max_pages=1 << 26)), "keys")
    refused(attention(cache(tokens=1 << 29, offsets=64)), "large")
    # (2^24 workgroups of 256 threads are more than a launch takes)
    refused(attention(cache(tokens=1 << 24, batch=1 << 24), workspace=P, nbytes=1 << 62), "large")
    for scale in (float("nan"), float("inf"), 3e38):
        refused(attention(cache(), scale=scale), "scale")
    refused(attention(cache(), length=50), "workspace")
    refused(attention(cache(), length=50, workspace=P, nbytes=workspace_bytes(cache(), length=50) - 1), "workspace")
    refused(attention(cache(), length=50, workspace=ctypes.c_void_p(72), nbytes=1 << 30), "workspace", "aligned")
    assert attention(cache(tokens=0, batch=0)) == 0
    assert workspace_bytes(cache(page_size=8)) == -1 and "page_size" in _kernels.last_error()
    assert workspace_bytes(cache(tokens=0, batch=0)) == 0
    # one part of a row: (m, l) and head_dim numbers in 32 bits
    assert workspace_bytes(cache(), length=16) % (3 * 4 * (64 * 4 + 8)) == 0 < workspace_bytes(cache(), length=16)


def test_eager_calls_take_gpu_tensors_only():
    x = torch.zeros(2, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        eager.quantize_rows(x)
    with pytest.raises(ValueError, match="GPU"):
        eager.gemm_rcr_int8(x.to(torch.int8), x.to(torch.int8), x.float(), x.float())
    with pytest.raises(ValueError, match="GPU"):
        eager.rotary_embedding(x, torch.zeros(2, dtype=torch.int64), torch.zeros(32))
    with pytest.raises(ValueError, match="GPU"):
        eager.paged_kv_append(x, x, x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        eager.prefix_attention(x, x, x, x, x)


def test_frequencies():
    freqs, scale = eager.rotary_frequencies(64, device="cpu")
    want = 10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / -64)
    assert scale == 1.0 and freqs.dtype == torch.float32 and torch.equal(freqs, want.float())
    assert torch.equal(eager.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")[0], (want / 4).float())
    # the base raised: the highest frequency stays, the lowest is divided by the factor
    raised, _ = eager.rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert raised[0] == 1.0 and abs(raised[-1].item() / (want[-1].item() / 4) - 1) < 1e-6
    for scaling in ("bands", "yarn"):
        got, scale = eager.rotary_frequencies(128, base=500000.0, scaling=scaling, factor=8.0, original_length=8192, low=1.0, high=4.0,
                                              device="cpu")
        plain = 500000.0 ** (torch.arange(0, 128, 2, dtype=torch.float64) / -128)
        turns = 8192 * plain / (2 * math.pi)
        share = (got.double() / plain - 1 / 8) / (1 - 1 / 8)
        # (yarn's bounds are whole pairs, rounded outwards)
        edge = 1e-6
        assert (share >= -edge).all() and (share <= 1 + edge).all() and (share[1:] <= share[:-1] + edge).all()
        slow, fast = torch.nonzero(turns < 1.0)[:, 0], torch.nonzero(turns > 4.0)[:, 0]
        assert (share[slow[1:]].abs() < edge).all() and ((share[fast[:-1]] - 1).abs() < edge).all()
        assert abs(scale - (1.0 if scaling == "bands" else 0.1 * math.log(8.0) + 1.0)) < 1e-12


@pytest.mark.parametrize("arguments", [dict(rotated=63), dict(rotated=0), dict(rotated=64, scaling="other"), dict(rotated=64, base=1.0),
                                       dict(rotated=64, scaling="linear", factor=0.5), dict(rotated=64, scaling="yarn", factor=2.0),
                                       dict(rotated=2, scaling="base", factor=2.0),
                                       dict(rotated=64, scaling="bands", factor=2.0, original_length=2048, low=4.0, high=4.0)])
def test_frequencies_refused(arguments):
    with pytest.raises(ValueError):
        eager.rotary_frequencies(device="cpu", **arguments)
