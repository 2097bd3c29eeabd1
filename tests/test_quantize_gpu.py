"""Rows to 8-bit integers on the GPU: the integers are those of exact arithmetic, the scale is rounded once."""
import math

import pytest
import torch

from aitemplate_amd import eager

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(x, q, scale):
    most = x.double().abs().amax(-1, keepdim=True)
    # (127 x and the division are exact enough in 64 bits: see the kernel's comment, with 29 more bits)
    want = (x.double() * 127.0 / most).nan_to_num(0.0).round()
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == x.shape[:-1]
    assert torch.equal(q.double(), want)
    assert torch.equal(scale, (most[..., 0] / 127.0).float())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 7), (1, 64), (5, 511), (9, 512), (6, 520), (7, 1024), (2, 1025), (3, 2048), (5, 2056),
                                          (64, 4096), (3, 4097), (2, 8192), (3, 8199), (2, 16384), (2, 16385), (3, 40001)])
def test_rows(dtype, rows, columns):
    g = torch.Generator(device=DEV).manual_seed(rows * columns)
    x = torch.randn(rows, columns, device=DEV, generator=g) * torch.rand(rows, 1, device=DEV, generator=g).mul_(8).exp2()
    x = x.to(dtype)
    check(x, *eager.quantize_rows(x))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_value_against_every_maximum(dtype):
    # all positive values next to middles of whole numbers: every mantissa against some maxima, ties among them
    bits = torch.arange(1, 0x7c00 if dtype == torch.float16 else 0x7f80, device=DEV, dtype=torch.int32)
    for most in (254.0, 127.0, 1.0, 3.0, 0.0078125, 200.0, 65504.0):
        m = torch.tensor(most, device=DEV).to(dtype)
        v = bits.to(torch.int16).view(dtype)
        v = v[(v <= m) & (v >= m / 4096)]
        x = torch.cat((m[None], v, -v)).view(1, -1).contiguous()
        check(x, *eager.quantize_rows(x))


@pytest.mark.parametrize("columns", [40, 3000, 20000])
def test_the_largest_and_smallest_numbers(columns):
    # 127 times the largest bfloat16 is beyond 32-bit floats
    g = torch.Generator(device=DEV).manual_seed(columns)
    x = (torch.rand(8, columns, device=DEV, generator=g) * 2 - 1).bfloat16()
    x *= torch.tensor([2.0 ** e for e in (127, 126, 121, 120, 101, 100, -100, -120)], device=DEV)[:, None].bfloat16()
    x[0, 3], x[0, 5] = torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).min
    check(x, *eager.quantize_rows(x))
    x = torch.full((2, columns), torch.finfo(torch.float16).max, device=DEV, dtype=torch.float16)
    x[1, ::2] = 2.0 ** -24
    check(x, *eager.quantize_rows(x))


def test_shapes_pitch_and_places():
    x = torch.randn(3, 5, 96, device=DEV).half()
    q, s = eager.quantize_rows(x)
    check(x, q, s)
    wide = torch.randn(6, 200, device=DEV).bfloat16()
    view = wide[:, 3:100]
    check(view, *eager.quantize_rows(view))
    q, s = torch.full((6, 97), 99, dtype=torch.int8, device=DEV), torch.full((6,), -1.0, device=DEV)
    got = eager.quantize_rows(view, out=q, scale=s)
    assert got[0] is q and got[1] is s
    check(view, q, s)
    q, s = eager.quantize_rows(torch.empty(0, 16, device=DEV).half())
    assert q.shape == (0, 16) and s.shape == (0,)
    q, s = eager.quantize_rows(torch.empty(3, 0, device=DEV).half())
    assert q.shape == (3, 0) and torch.equal(s, torch.zeros(3, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("columns", [40, 3000, 20000])
def test_rows_of_zeros_infinities_and_nan(dtype, columns):
    x = torch.randn(6, columns, device=DEV).to(dtype)
    x[1] = 0.0
    x[2, 17], x[3, columns - 1], x[4, 0] = math.inf, math.nan, -math.inf
    x[5] = torch.finfo(dtype).tiny * 2.0 ** -3  # a subnormal row
    q, s = eager.quantize_rows(x)
    ok = torch.tensor([0, 1, 5], device=DEV)
    check(x[ok], q[ok], s[ok])
    assert s[1] == 0 and torch.isnan(s[2:5]).all() and not q[1:5].any()


def test_more_rows_than_one_launch_takes():
    # (2^24 workgroups of 16 rows and one more)
    x = torch.ones((1 << 28) + 5, 1, dtype=torch.float16, device=DEV)
    q, s = eager.quantize_rows(x)
    assert (q == 127).all() and (s == 1 / torch.tensor(127.0, device=DEV)).all()


def test_captured_and_replayed():
    x = torch.randn(64, 4096, device=DEV).half()
    q, s = eager.quantize_rows(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eager.quantize_rows(x, out=q, scale=s)
    for _ in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check(x, q, s)
