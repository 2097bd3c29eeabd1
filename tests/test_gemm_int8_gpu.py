"""Products of 8-bit integers with scales on the GPU, against 64 bits.

Tolerance: the sum is exact; it, the product of the scales, their product and the sum with the bias are rounded to 32 bits
(2^-24 relative each, the last of the result), the result once to its type: eps / 2 |y|, or half of its smallest number."""
import ctypes

import pytest
import torch

from aitemplate_amd import _kernels, eager

pytestmark = pytest.mark.gpu
DEV = "cuda"


def inputs(M, N, K, dtype, seed=0, bias=True):
    g = torch.Generator(device=DEV).manual_seed(seed + M * 7 + N * 3 + K)
    a, b = (torch.randint(-128, 128, (n, K), device=DEV, generator=g, dtype=torch.int8) for n in (M, N))
    a_scale, b_scale = (torch.rand(n, device=DEV, generator=g).add_(0.1).mul_(0.01) for n in (M, N))
    return a, b, a_scale, b_scale, torch.randn(N, device=DEV, generator=g).to(dtype) if bias else None


def check(got, a, b, a_scale, b_scale, bias):
    dtype = got.dtype
    scaled = (a.double() @ b.double().t()) * a_scale.double()[:, None] * b_scale.double()
    want = scaled if bias is None else scaled + bias.double()
    info = torch.finfo(dtype)
    allowed = (want.abs() * (info.eps / 2 + 2.0 ** -24) + scaled.abs() * 3 * 2.0 ** -24) * (1 + 1e-4) + info.smallest_normal * info.eps / 2
    assert got.shape == want.shape
    worst = ((got.double() - want).abs() / allowed).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst


SIZES = [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (3, 5, 7), (16, 16, 64), (17, 33, 48), (4, 1000, 2048), (33, 70, 100), (64, 64, 1024),
         (64, 512, 4096), (100, 130, 260), (130, 260, 130), (255, 257, 255), (256, 256, 512), (300, 1000, 1101), (512, 512, 64), (513, 776, 1040),
         (1024, 768, 768), (2000, 1024, 272), (2048, 2304, 16), (777, 2731, 1101), (1000, 4096, 514), (5, 8, 131071)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(dtype, bias, M, N, K):
    x = inputs(M, N, K, dtype, bias=bias)
    check(eager.gemm_rcr_int8(*x, dtype=dtype), *x)
    need = eager.gemm_int8_workspace_bytes(M, N, K, bias, dtype)
    check(eager.gemm_rcr_int8(*x, dtype=dtype, workspace=eager.new_workspace(need)), *x)


def instances(dtype, bias):
    return _kernels.gemm_algo_names(1 if bias else 0, 2 + (dtype == torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_every_instance(dtype, bias):
    lib = _kernels.load()
    names, ran = instances(dtype, bias), set()
    for M, N, K in [(130, 264, 592), (600, 520, 1104), (40, 2048, 4096), (257, 385, 516), (300, 776, 1036), (70, 96, 96)]:
        x = inputs(M, N, K, dtype, bias=bias)
        for i, name in enumerate(names):
            if not lib.aitamd_gemm_algo_supported(int(bias), 2 + (dtype == torch.bfloat16), i, M, N, K // 2, K // 2, K // 2, 16 if K % 16 == 0 else 4):
                continue
            need = eager.gemm_int8_workspace_bytes(M, N, K, bias, dtype, algo=i)
            got = eager.gemm_rcr_int8(*x, dtype=dtype, algo=i, workspace=eager.new_workspace(need) if need else None)
            try:
                check(got, *x)
            except AssertionError as e:
                raise AssertionError(f"{name} {M} x {N} x {K}: {e}")
            ran.add(name)
    assert ran == set(names)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_largest_sums(dtype):
    # the largest magnitudes of both signs, at the longest K: sums of +- 2^31 - 2^14
    for K, instance in ((131071, None), (131068, None), (131056, None)):
        a, b = torch.full((20, K), -128, dtype=torch.int8, device=DEV), torch.full((24, K), -128, dtype=torch.int8, device=DEV)
        b[::2] = 127
        a_scale, b_scale = torch.full((20,), 1e-4, device=DEV), torch.full((24,), 1e-4, device=DEV)
        check(eager.gemm_rcr_int8(a, b, a_scale, b_scale, dtype=dtype), a, b, a_scale, b_scale, None)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_pitches_addresses_and_places(dtype):
    for M, N, K, start, wide in [(70, 96, 128, 16, 160), (70, 96, 128, 4, 148), (70, 96, 128, 1, 151), (70, 97, 101, 0, 128), (1, 96, 100, 3, 103)]:
        a, b, a_scale, b_scale, bias = inputs(M, N, K, dtype)
        hold = [torch.full((n * wide + start,), 77, dtype=torch.int8, device=DEV) for n in (M, N)]
        a2, b2 = (t[start:].view(n, wide)[:, :K] for t, n in zip(hold, (M, N)))
        a2.copy_(a), b2.copy_(b)
        check(eager.gemm_rcr_int8(a2, b2, a_scale, b_scale, bias, dtype=dtype), a, b, a_scale, b_scale, bias)
        # into rows of a wider buffer, at an odd element
        out = torch.full((M * (N + 5) + 1,), 3.0, dtype=dtype, device=DEV)
        view = out[1:].view(M, N + 5)[:, :N]
        assert eager.gemm_rcr_int8(a, b, a_scale, b_scale, bias, dtype=dtype, out=view) is view
        check(view, a, b, a_scale, b_scale, bias)
        assert out[0] == 3.0 and (out[1:].view(M, N + 5)[:, N:] == 3.0).all()
    x = inputs(6, 40, 64, dtype)
    got = eager.gemm_rcr_int8(x[0].view(2, 3, 64), x[1], x[2].view(2, 3), *x[3:], dtype=dtype)
    assert got.shape == (2, 3, 40)
    check(got.view(6, 40), *x)


def test_rows_far_apart():
    # 8 MiB from row to row: further than a tile's 32-bit offsets reach
    M, N, K, pitch = 300, 70, 128, 1 << 23
    a, b, a_scale, b_scale, bias = inputs(M, N, K, torch.float16)
    hold = torch.zeros(M * pitch, dtype=torch.int8, device=DEV)
    far = hold.as_strided((M, K), (pitch, 1))
    far.copy_(a)
    check(eager.gemm_rcr_int8(far, b, a_scale, b_scale, bias), a, b, a_scale, b_scale, bias)


def test_nothing_to_sum_and_nothing_to_write():
    a, b, a_scale, b_scale, bias = inputs(5, 8, 0, torch.float16)
    assert torch.equal(eager.gemm_rcr_int8(a, b, a_scale, b_scale, bias), bias.expand(5, 8))
    assert not eager.gemm_rcr_int8(a, b, a_scale, b_scale).any()
    a, b, a_scale, b_scale, bias = inputs(0, 8, 16, torch.float16)
    assert eager.gemm_rcr_int8(a, b, a_scale, b_scale, bias).shape == (0, 8)


def test_rows_without_a_scale():
    # a NaN scale (a quantized row that held an infinity) is its row's only; a zero scale gives the bias
    a, b, a_scale, b_scale, bias = inputs(40, 64, 128, torch.float16)
    a_scale[3], a_scale[7] = float("nan"), 0.0
    got = eager.gemm_rcr_int8(a, b, a_scale, b_scale, bias)
    assert torch.isnan(got[3]).all() and torch.equal(got[7], bias)
    keep = torch.tensor([i for i in range(40) if i != 3], device=DEV)
    check(got[keep], a[keep], b, a_scale[keep], b_scale, bias)


def test_quantized_layer():
    # a layer in 8 bits: quantized rows times a quantized weight, next to the layer itself.  An element of x is off by half of
    # max|x| / 127 at most, one of w likewise, so a product's sum by K of those, and the product of both
    x, w = torch.randn(33, 512, device=DEV).half(), (torch.randn(96, 512, device=DEV) * 512 ** -0.5).half()
    got = eager.gemm_rcr_int8(*[t for pair in zip(eager.quantize_rows(x), eager.quantize_rows(w)) for t in pair])
    want = x.double() @ w.double().t()
    dx, dw = (t.double().abs().amax(1, keepdim=True) / 254 for t in (x, w))
    allowed = dx * w.double().abs().sum(1) + x.double().abs().sum(1, keepdim=True) * dw.t() + 512 * dx * dw.t() + want.abs() * 2.0 ** -10
    assert ((got.double() - want).abs() <= allowed + 1e-3 * allowed).all()


def test_captured_and_replayed():
    for M, N, K in [(64, 512, 4096), (7, 33, 65)]:
        a, b, a_scale, b_scale, bias = inputs(M, N, K, torch.float16)
        workspace = eager.new_workspace(eager.gemm_int8_workspace_bytes(M, N, K, True))
        out = torch.empty(M, N, dtype=torch.float16, device=DEV)

        def step():
            return eager.gemm_rcr_int8(a, b, a_scale, b_scale, bias, out=out, workspace=workspace)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for k in range(4):
            a.random_(-128, 128)
            graph.replay()
            torch.cuda.synchronize()
            check(out, a, b, a_scale, b_scale, bias)
