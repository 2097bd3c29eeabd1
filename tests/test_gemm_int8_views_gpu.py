"""Products of 8-bit integers whose K is a multiple of 4 and whose operands are views off dword addresses: the one, the other or
both are laid out in scratch memory first, which the calls without a workspace allocate and the size query knows.  Tolerance: see
test_gemm_int8_gpu.py."""
import pytest
import torch

from aitemplate_amd import _kernels, eager
from test_gemm_int8_gpu import DEV, check, inputs

pytestmark = pytest.mark.gpu


def view(t, start, pitch):
    """The rows of t at byte `start`, `pitch` bytes apart, between bytes that do not belong to them."""
    rows, columns = t.shape
    hold = torch.full((start + rows * pitch,), 77, dtype=torch.int8, device=DEV)
    v = hold[start:].view(rows, pitch)[:, :columns]
    v.copy_(t)
    return v


PLACES = {"pitch": lambda t: view(t, 0, t.shape[1] + 1), "address": lambda t: view(t, 3, t.shape[1]), "both": lambda t: view(t, 1, t.shape[1] + 6),
          "dwords": lambda t: view(t, 4, t.shape[1] + 12)}
CASES = [(a, b) for a in PLACES for b in PLACES if (a, b) != ("dwords", "dwords")]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("place_a,place_b", CASES)
@pytest.mark.parametrize("M,N,K", [(1, 96, 1024), (64, 520, 516), (130, 257, 1040), (300, 70, 512), (33, 64, 4096)])
def test_views(dtype, place_a, place_b, M, N, K):
    a, b, *rest = inputs(M, N, K, dtype)
    at = PLACES[place_a](a), PLACES[place_b](b)
    check(eager.gemm_rcr_int8(*at, *rest, dtype=dtype), a, b, *rest)
    check(eager.gemm_rcr_int8(*at, *rest[:2], dtype=dtype), a, b, *rest[:2], None)
    need = eager.gemm_int8_workspace_bytes(M, N, K, True, dtype, any_byte=True)
    assert need >= 4096 + (M + N) * K or K <= 512  # (at 512 and less only what the instances that share tiles take)
    for size in {need, max(need - 16 * (M + N), 0), 4096}:  # (too little: as the rows lie)
        workspace = torch.zeros(size, dtype=torch.uint8, device=DEV)
        check(eager.gemm_rcr_int8(*at, *rest, dtype=dtype, workspace=workspace), a, b, *rest)
        assert not workspace[:4096].any()


@pytest.mark.parametrize("python_only", [False, True])
@pytest.mark.parametrize("place_a,place_b", CASES)
def test_scratch_memory_is_allocated(place_a, place_b, python_only, monkeypatch):
    if python_only:
        monkeypatch.setattr(eager, "_native_decoder", _kernels._NoNative())
    M, N, K = 256, 512, 2048
    a, b, *rest = inputs(M, N, K, torch.float16)
    at = PLACES[place_a](a), PLACES[place_b](b)
    eager.gemm_rcr_int8(*at, *rest)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    eager.gemm_rcr_int8(*at, *rest)
    used = torch.cuda.max_memory_allocated() - before - M * N * 2
    # (a row that is alone has no pitch)
    want = (M * K if place_a != "dwords" else 0) + (N * K if place_b != "dwords" else 0)
    assert want <= used <= want + 4096 + 4096


def test_whole_dwords_take_none():
    a, b, *rest = inputs(256, 512, 2048, torch.float16)
    eager.gemm_rcr_int8(a, b, *rest)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    eager.gemm_rcr_int8(a, b, *rest)
    assert torch.cuda.max_memory_allocated() - before <= 256 * 512 * 2


def test_captured_and_replayed():
    M, N, K = 70, 96, 1024
    a, b, *rest = inputs(M, N, K, torch.float16)
    at = PLACES["pitch"](a), PLACES["dwords"](b)
    workspace = eager.new_workspace(eager.gemm_int8_workspace_bytes(M, N, K, True, any_byte=True))
    out = torch.empty(M, N, dtype=torch.float16, device=DEV)
    eager.gemm_rcr_int8(*at, *rest, out=out, workspace=workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eager.gemm_rcr_int8(*at, *rest, out=out, workspace=workspace)
    for _ in range(3):
        at[0].random_(-128, 128)
        graph.replay()
        torch.cuda.synchronize()
        check(out, at[0].contiguous(), b, *rest)
