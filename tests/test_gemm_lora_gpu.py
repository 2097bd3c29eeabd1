"""A shared projection with the low-rank adapters of its rows, on the GPU, against 64 bits.

Tolerance, element by element: the result's rounding (half a step of its type, eps / 2 relative, at least half the smallest step);
sums in 32 bits, of n numbers off by at most n 2^-24 of the sum of their magnitudes, over K and the ranks; the adapters' sums over K
likewise, and held within 2^-17 of themselves."""
import pytest
import torch

from aitemplate_amd import _kernels, eager

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(dtype, M, N, K, rank, n, seed=0, bias=False, scales=True):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)

    return dict(x=normal(M, K), w=normal(N, K, scale=max(K, 1) ** -0.5), lora_a=normal(n, rank, K, scale=max(K, 1) ** -0.5),
                lora_b=normal(n, N, rank, scale=rank ** -0.5), adapters=torch.randint(-1, n + 1, (M,), device=DEV, generator=g, dtype=torch.int32),
                scales=torch.rand(n, device=DEV, generator=g) + 0.5 if scales else None, bias=normal(N) if bias else None)


def expected(x, w, lora_a, lora_b, adapters, scales=None, bias=None):
    """The result in 64 bits, and what it may be off by ahead of its rounding."""
    x, n = x.double(), lora_a.shape[0]
    wt = w.double().t()
    y, size = x @ wt, x.abs() @ wt.abs()
    steps = (x.shape[1] + lora_a.shape[1] + 8) * 2.0 ** -24
    held = torch.zeros_like(y)
    for i in range(n):
        rows = (adapters == i).nonzero()[:, 0]
        if len(rows) == 0:
            continue
        a, b = lora_a[i].double().t(), lora_b[i].double().t()
        s = 1.0 if scales is None else scales[i].double()
        t = s * (x[rows] @ a)
        y[rows] += t @ b
        size[rows] += abs(s) * (x[rows].abs() @ a.abs()) @ b.abs()
        held[rows] += t.abs() @ b.abs() * 2.0 ** -17
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size * steps + held


def check(got, args):
    want, off = expected(**args)
    info = torch.finfo(got.dtype)
    allowed = (want.abs() + off) * info.eps / 2 + off + info.smallest_normal * info.eps / 2
    worst = ((got.double() - want).abs() / allowed).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst


SIZES = [(1, 64, 64, 8, 1), (1, 4096, 1024, 16, 3), (3, 33, 17, 1, 2), (16, 256, 128, 16, 5), (33, 130, 200, 12, 4), (64, 520, 512, 32, 40),
         (65, 96, 1030, 7, 3), (257, 264, 320, 24, 3), (300, 1000, 513, 20, 2), (513, 512, 640, 64, 6), (700, 768, 192, 130, 3),
         (1000, 48, 4096, 16, 7), (2100, 2048, 256, 16, 5), (40, 8, 3000, 1024, 2), (31, 1, 9, 3, 1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K,rank,n", SIZES)
def test_mixed_rows(dtype, M, N, K, rank, n):
    args = make(dtype, M, N, K, rank, n, seed=M + N, bias=(M + N) % 2 == 0, scales=rank != 8)
    check(eager.gemm_rcr_lora(**args), args)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K,rank", [(2, 64, 256, 16), (130, 264, 512, 16), (600, 512, 256, 40), (1500, 2304, 512, 9)])
def test_requests_in_a_row(dtype, M, N, K, rank):
    args = make(dtype, M, N, K, rank, 5, seed=M, bias=True)
    cuts = [0, M // 5, M // 3, M // 3 + 1, M - 1, M]
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        args["adapters"][a:b] = (3, -1, 0, 3, 99)[i]
    check(eager.gemm_rcr_lora(**args), args)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_every_instance(dtype, bias):
    """All tiles, at sizes that they all take, with one adapter, with a few and with many among a wave's rows."""
    d = 0 if dtype is torch.float16 else 1
    args = make(dtype, 400, 520, 640, 24, 60, bias=bias)
    for which in ("one", "few", "many"):
        rows = torch.arange(400, device=DEV)
        args["adapters"] = {"one": torch.full((400,), 7, device=DEV), "few": rows // 9 % 4 - 1, "many": rows * 7 % 61 - 1}[which].int()
        for i, name in enumerate(_kernels.gemm_algo_names(int(bias), 4 + d)):
            print(name, which, flush=True)
            check(eager.gemm_rcr_lora(**args, algo=i), args)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_without_adapters_it_is_the_plain_product(dtype):
    args = make(dtype, 50, 264, 320, 16, 3, bias=True)
    args["adapters"].fill_(-1)
    args["lora_a"].fill_(float("nan")), args["lora_b"].fill_(float("inf"))
    got = eager.gemm_rcr_lora(**args)
    info, want, off = torch.finfo(dtype), *expected(**args)
    assert ((got.double() - want).abs() <= (want.abs() + off) * info.eps / 2 + off).all()
    # ... nor do other rows' adapters matter to one
    args["adapters"][7] = 1
    again = eager.gemm_rcr_lora(**args)
    others = torch.arange(50, device=DEV) != 7
    assert torch.equal(again[others], got[others]) and not again[7].isfinite().any()


def test_views_leading_dims_and_pitch():
    args = make(torch.float16, 24, 96, 128, 16, 3, bias=True)
    want = eager.gemm_rcr_lora(**args)
    wide = torch.full((24, 200), float("nan"), device=DEV).half()
    wide[:, 3:131] = args["x"]
    w = torch.full((96, 130), float("nan"), device=DEV).half()
    w[:, 1:129] = args["w"]
    out = torch.zeros(24, 110, device=DEV).half()
    got = eager.gemm_rcr_lora(**{**args, "x": wide[:, 3:131], "w": w[:, 1:129], "out": out[:, 5:101]})
    check(got, args)
    assert (out[:, :5] == 0).all() and (out[:, 101:] == 0).all()
    lead = eager.gemm_rcr_lora(**{**args, "x": args["x"].view(2, 12, 128), "adapters": args["adapters"].view(2, 12)})
    assert lead.shape == (2, 12, 96) and torch.equal(lead.view(24, 96), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-6, 300.0])
@pytest.mark.parametrize("M", [5, 600])
def test_sums_beyond_a_halfs_range(dtype, size, M):
    """Adapters whose sums over K are far above 65504 or far below a half's steps, and come back into its range."""
    args = make(dtype, M, 72, 512, 16, 2, scales=False)
    args["adapters"].fill_(1)
    args["lora_a"] = (args["lora_a"].float() * 512 ** 0.5 * (size if size > 1 else 1)).to(dtype)
    args["scales"] = torch.full((2,), size if size > 1 else size ** 2, device=DEV)
    args["lora_b"] = (args["lora_b"].float() * (1e-4 if size > 1 else 60.0)).to(dtype)
    args["w"] *= 0
    check(eager.gemm_rcr_lora(**args), args)


def test_empty():
    args = make(torch.float16, 4, 16, 32, 8, 2, bias=True)
    assert eager.gemm_rcr_lora(**{**args, "x": args["x"][:0], "adapters": args["adapters"][:0]}).shape == (0, 16)
    none = eager.gemm_rcr_lora(**{**args, "lora_a": args["lora_a"][:0], "lora_b": args["lora_b"][:0], "scales": args["scales"][:0]})
    assert torch.equal(none, eager.gemm("gemm_rcr_bias", args["x"], args["w"], args["bias"]))
    no_k = make(torch.bfloat16, 300, 16, 0, 8, 2, bias=True)
    assert torch.equal(eager.gemm_rcr_lora(**no_k), no_k["bias"].expand(300, 16))


def test_workspace_of_a_callers_own_and_captured():
    args = make(torch.bfloat16, 64, 1536, 2048, 16, 20)
    need = eager.gemm_lora_workspace_bytes(64, 1536, 2048, 16, dtype=torch.bfloat16)
    ws = torch.full((need + 32,), 255, dtype=torch.uint8, device=DEV)
    want = eager.gemm_rcr_lora(**args)
    out = torch.empty_like(want)
    eager.gemm_rcr_lora(**args, out=out, workspace=ws[:need])
    assert torch.equal(out, want) and (ws[need:] == 255).all() and (ws[:4096] == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eager.gemm_rcr_lora(**args, out=out, workspace=ws[:need])
    for step in range(4):
        args["x"].copy_(torch.randn_like(args["x"]))
        args["adapters"].copy_(torch.randint_like(args["adapters"], -1, 20))
        ws.fill_(step * 77)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager.gemm_rcr_lora(**args))


def test_refusals():
    args = make(torch.float16, 4, 16, 32, 8, 2)
    for changed, word in (({"lora_a": args["lora_a"][:, :, :16]}, "lora_a"), ({"lora_b": args["lora_b"][:1]}, "lora_b"),
                          ({"adapters": args["adapters"].long()}, "adapters"), ({"adapters": args["adapters"][:3]}, "adapters"),
                          ({"scales": args["scales"][:1]}, "scales"), ({"w": args["w"].bfloat16()}, "w"), ({"x": args["x"].float()}, "x"),
                          ({"out": torch.empty(4, 15, device=DEV).half()}, "out"), ({"x": args["x"].cpu()}, "x")):
        with pytest.raises(ValueError, match=word):
            eager.gemm_rcr_lora(**{**args, **changed})
    with pytest.raises(RuntimeError, match="workspace"):
        eager.gemm_rcr_lora(**args, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError, match="range"):
        eager.gemm_rcr_lora(**args, algo=999)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank", [1, 8, 31, 33, 64, 65, 130])
@pytest.mark.parametrize("M,N,K", [(64, 1536, 4096), (29, 2056, 2272), (200, 512, 2048), (129, 300, 4100)])
def test_tiles_that_share_k(dtype, M, N, K, rank):
    """Few tiles with a long K, whose adapters are split among workgroups: almost every row with its own, or all with one."""
    args = make(dtype, M, N, K, rank, 50, seed=rank)
    check(eager.gemm_rcr_lora(**args), args)
    args["adapters"].fill_(49)
    check(eager.gemm_rcr_lora(**args), args)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [7, 64, 700, 2100])
def test_a_row_that_is_no_numbers_is_alone(dtype, M):
    args = make(dtype, M, 1024, 512, 16, 6, seed=M)
    want = eager.gemm_rcr_lora(**args)
    args["x"][M // 2, 5], args["x"][M - 1, 500] = float("nan"), float("inf")
    got = eager.gemm_rcr_lora(**args)
    others = torch.ones(M, dtype=torch.bool, device=DEV)
    others[M // 2] = others[M - 1] = False
    assert torch.equal(got[others], want[others]) and not torch.isfinite(got[~others]).any()
