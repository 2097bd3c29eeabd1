"""A compiled model whose run brings offsets that do not fit its sequences: an error from the host, nothing launched, and the next run
with fitting ones is right."""
import pytest
import torch

from aitemplate_amd import eager
from aitemplate_amd.compiler import ops
from aitemplate_amd.frontend import IntImm, IntVar
from paged_common import DEV, Paged
from test_decoder_graph_gpu import build, feed

pytestmark = pytest.mark.gpu


def test_offsets_of_another_batch():
    H, C, D, page = 4, 2, 64, 16
    c = Paged(torch.float16, [20, 3, 40], [5, 1, 9], C, D, page, ragged=True)
    T, B, P = IntVar(values=[1, 64], name="tokens"), IntVar(values=[1, 8], name="sequences"), IntVar(values=[1, 64], name="pages")
    q, k, v = (feed(n, [T, IntImm(h), IntImm(D)], "float16") for n, h in (("q", H), ("k", C), ("v", C)))
    k_cache, v_cache = (feed(n, [P, IntImm(page), IntImm(C), IntImm(D)], "float16") for n in ("k_cache", "v_cache"))
    table, lengths = feed("table", [B, IntVar(values=[1, 16], name="most")], "int32"), feed("lengths", [B], "int32")
    freqs, offsets = feed("freqs", [IntImm(D // 2)], "float32"), feed("offsets", [IntVar(values=[2, 9], name="ends")], "int32")
    turned = ops.paged_kv_append()(q, k, v, k_cache, v_cache, table, lengths, freqs, offsets)
    module = build([ops.prefix_attention()(turned, k_cache, v_cache, table, lengths, offsets)])
    rows = torch.randn(c.tokens, H + 2 * C, D, device=DEV).half()
    ins = {"q": rows[:, :H].contiguous(), "k": rows[:, H:H + C].contiguous(), "v": rows[:, H + C:].contiguous(), "k_cache": c.k, "v_cache": c.v,
           "table": c.table, "lengths": c.lengths, "freqs": eager.rotary_frequencies(D, device=DEV)[0], "offsets": c.offsets}
    before = [t.clone() for t in (c.k, c.v)]
    out = torch.full((c.tokens, H, D), 9.0, device=DEV, dtype=torch.float16)
    for wrong in (c.offsets[:2], c.offsets[:3], torch.cat((c.offsets, c.offsets[-1:]))):
        with pytest.raises(RuntimeError):
            module.run_with_tensors({**ins, "offsets": wrong.contiguous()}, [out])
        torch.cuda.synchronize()
        assert (out == 9.0).all() and all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip((c.k, c.v), before))
    module.run_with_tensors(ins, [out])
    turned = eager.paged_kv_append(ins["k"], ins["v"], c.k, c.v, c.table, c.lengths, c.offsets, q=ins["q"], freqs=ins["freqs"])
    assert torch.equal(out, eager.prefix_attention(turned, c.k, c.v, c.table, c.lengths, c.offsets))
