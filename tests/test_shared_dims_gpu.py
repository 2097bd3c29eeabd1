"""Inputs of a compiled model that share a dimension have to agree on it at a run: an error from the host, nothing launched."""
import pytest
import torch

from aitemplate_amd import eager
from aitemplate_amd.compiler import ops
from aitemplate_amd.frontend import IntImm, IntVar
from paged_common import DEV, Paged
from test_decoder_graph_gpu import build, feed

pytestmark = pytest.mark.gpu


def test_paged_attention():
    H, C, D, page = 4, 2, 64, 16
    c = Paged(torch.float16, [20, 3, 40], [1, 1, 1], C, D, page)
    B, P = IntVar(values=[1, 8], name="sequences"), IntVar(values=[1, 64], name="pages")
    q = feed("q", [B, IntImm(H), IntImm(D)], "float16")
    k_cache, v_cache = (feed(n, [P, IntImm(page), IntImm(C), IntImm(D)], "float16") for n in ("k_cache", "v_cache"))
    table, lengths = feed("table", [B, IntVar(values=[1, 16], name="most")], "int32"), feed("lengths", [B], "int32")
    module = build([ops.prefix_attention()(q, k_cache, v_cache, table, lengths)])
    rows = torch.randn(3, H, D, device=DEV).half()
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    ins = {"q": rows, "k_cache": c.k, "v_cache": c.v, "table": c.table, "lengths": c.lengths}
    out = torch.full((3, H, D), 9.0, device=DEV, dtype=torch.float16)
    for wrong in ({"table": c.table[:2].contiguous()}, {"lengths": c.lengths[:1].contiguous()}, {"q": rows[:2].contiguous()},
                  {"v_cache": c.v[:2].contiguous()}, {"table": c.table[:2].contiguous(), "q": rows[:2].contiguous()}):
        for names in (list(ins), list(ins)[::-1]):
            with pytest.raises(RuntimeError):
                module.run_with_tensors({n: {**ins, **wrong}[n] for n in names}, [out])
        torch.cuda.synchronize()
        assert (out == 9.0).all()
    module.run_with_tensors(ins, [out])
    assert torch.equal(out, eager.prefix_attention(rows, c.k, c.v, c.table, c.lengths))


def test_gemm_with_a_residual():
    M = IntVar(values=[1, 64], name="M")
    x, d = feed("x", [M, IntImm(64)], "float16"), feed("d", [M, IntImm(32)], "float16")
    w, b = feed("w", [IntImm(32), IntImm(64)], "float16"), feed("b", [IntImm(32)], "float16")
    module = build([ops.gemm_rcr_bias_add()(x, w, b, d)])
    xt, dt, wt, bt = (torch.randn(*s, device=DEV).half() for s in ((20, 64), (20, 32), (32, 64), (32,)))
    out = torch.empty(20, 32, device=DEV, dtype=torch.float16)
    for wrong in ({"d": dt[:5].contiguous()}, {"x": xt[:5].contiguous()}):
        with pytest.raises(RuntimeError):
            module.run_with_tensors({"x": xt, "w": wt, "b": bt, "d": dt, **wrong}, [out])
    module.run_with_tensors({"x": xt, "w": wt, "b": bt, "d": dt}, [out])
    assert torch.equal(out, eager.gemm("gemm_rcr_bias_add", xt, wt, bias=bt, d0=dt)) or torch.allclose(
        out.float(), xt.float() @ wt.float().t() + bt.float() + dt.float(), atol=2 ** -8, rtol=2 ** -10)
