"""The decoder operators as graph ops: graph -> compile_model() -> library -> run, against the eager calls (which have tests of
their own) and, for the whole block, against plain torch."""
import itertools
import os

import pytest
import torch

from aitemplate_amd import eager
from aitemplate_amd.compiler import compile_model, ops
from aitemplate_amd.frontend import IntImm, IntVar, Tensor
from aitemplate_amd.testing import detect_target
from paged_common import DEV, Paged

pytestmark = pytest.mark.gpu

WORKDIR = os.environ.get("AIT_TEST_WORKDIR", "/tmp/aitemplate_amd_tests")
_counter = itertools.count()


def build(outputs):
    for i, t in enumerate(outputs):
        t._attrs["name"], t._attrs["is_output"] = f"output_{i}", True
    return compile_model(list(outputs), detect_target(), WORKDIR, f"decoder_{next(_counter)}")


def feed(name, shape, dtype):
    return Tensor(shape=shape, dtype=dtype, name=name, is_input=True)


TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16}


@pytest.mark.parametrize("dtype,interleaved,inverse", [("float16", False, False), ("bfloat16", True, True)])
def test_rotary(dtype, interleaved, inverse):
    batch, seq = IntVar(values=[1, 4], name="batch"), IntVar(values=[1, 40], name="seq")
    x = feed("x", [batch, seq, IntImm(6), IntImm(64)], dtype)
    positions, freqs = feed("positions", [batch, seq], "int64"), feed("freqs", [IntImm(16)], "float32")
    module = build([ops.rotary_embedding(interleaved, 1.5, inverse)(x, positions, freqs)])
    for b, s in ((4, 40), (1, 7)):
        ins = {"x": torch.randn(b, s, 6, 64, device=DEV).to(TORCH[dtype]), "positions": torch.randint(0, 10000, (b, s), device=DEV),
               "freqs": eager.rotary_frequencies(32, device=DEV)[0]}
        out = torch.empty_like(ins["x"])
        module.run_with_tensors(ins, [out])
        assert torch.equal(out, eager.rotary_embedding(*ins.values(), interleaved=interleaved, scale=1.5, inverse=inverse))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("N,K,bias", [(96, 256, True), (130, 64, False), (33, 1030, True), (40, 700, False)])
def test_quantized_linear(dtype, N, K, bias):
    tokens = IntVar(values=[1, 70], name="tokens")
    x = feed("x", [tokens, IntImm(K)], dtype)
    w, w_scale = feed("w", [IntImm(N), IntImm(K)], "int8"), feed("w_scale", [IntImm(N)], "float32")
    b = [feed("b", [IntImm(N)], dtype)] if bias else []
    q, scale = ops.quantize_rows()(x)
    module = build([ops.gemm_rcr_int8(dtype)(q, w, scale, w_scale, *b)])
    wq, ws = eager.quantize_rows(torch.randn(N, K, device=DEV).to(TORCH[dtype]))
    bt = torch.randn(N, device=DEV).to(TORCH[dtype]) if bias else None
    for m in (70, 1, 33):
        xt = torch.randn(m, K, device=DEV).to(TORCH[dtype])
        out = torch.empty(m, N, device=DEV, dtype=TORCH[dtype])
        module.run_with_tensors({"x": xt, "w": wq, "w_scale": ws, **({"b": bt} if bias else {})}, [out])
        xq, xs = eager.quantize_rows(xt)
        assert torch.equal(out, eager.gemm_rcr_int8(xq, wq, xs, ws, bt, dtype=TORCH[dtype]))


@pytest.mark.parametrize("ragged", [False, True])
def test_decoder_attention_block(ragged):
    """x -> 8-bit projection -> rotation into the cache -> attention with a shared prefix -> 8-bit projection, twice, with the
    weights bound as constants and the cache as an input that the model writes."""
    H, C, D, hidden, page, prefix = 8, 2, 64, 320, 16, 70
    past, new = ([20, 3, 40], [5, 1, 9]) if ragged else ([20, 3, 40, 0], [1, 1, 1, 1])
    c = Paged(torch.float16, past, [n + 4 for n in new], C, D, page, prefix, ragged=True)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    tokens, batch = starts[-1], len(past)
    offsets = torch.tensor(starts, dtype=torch.int32, device=DEV) if ragged else None
    # (rows that see NaN places do not see them: fill them for the plain form's sake)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)

    T, B = IntVar(values=[1, 64], name="tokens"), IntVar(values=[1, 8], name="sequences")
    if not ragged:
        T = B
    x = feed("x", [T, IntImm(hidden)], "float16")
    freqs = feed("freqs", [IntImm(D // 2)], "float32")
    P = IntVar(values=[1, 64], name="pages")
    k_cache, v_cache = (feed(n, [P, IntImm(page), IntImm(C), IntImm(D)], "float16") for n in ("k_cache", "v_cache"))
    table, lengths = feed("table", [B, IntVar(values=[1, 16], name="most")], "int32"), feed("lengths", [B], "int32")
    prefix_table = feed("prefix_table", [IntVar(values=[1, 16], name="shared")], "int32")
    offs = feed("offsets", [IntVar(values=[2, 9], name="ends")], "int32") if ragged else None

    def linear(t, name, n, k):
        q, scale = ops.quantize_rows()(t)
        return ops.gemm_rcr_int8()(q, Tensor([IntImm(n), IntImm(k)], dtype="int8", name=name + "_w"), scale,
                                   Tensor([IntImm(n)], dtype="float32", name=name + "_s"), Tensor([IntImm(n)], dtype="float16", name=name + "_b"))

    qkv = linear(x, "qkv", (H + 2 * C) * D, hidden)
    q, k, v = ops.split()(qkv, [H * D, C * D, C * D], 1)
    q, k, v = (ops.reshape()(t, [T, n, D]) for t, n in ((q, H), (k, C), (v, C)))
    turned = ops.paged_kv_append(first_position=prefix)(q, k, v, k_cache, v_cache, table, lengths, freqs, offs)
    y = ops.prefix_attention(prefix_length=prefix)(turned, k_cache, v_cache, table, lengths, offs, prefix_table)
    module = build([linear(ops.reshape()(y, [T, H * D]), "out", hidden, H * D)])

    g = torch.Generator(device=DEV).manual_seed(3)
    w = {}
    for name, n, kk in (("qkv", (H + 2 * C) * D, hidden), ("out", hidden, H * D)):
        w[name + "_w"], w[name + "_s"] = eager.quantize_rows((torch.randn(n, kk, device=DEV, generator=g) * kk ** -0.5).half())
        w[name + "_b"] = torch.randn(n, device=DEV, generator=g).half() * 0.1
    module.set_many_constants_with_tensors(w)
    f, _ = eager.rotary_frequencies(D, device=DEV)
    for step in range(2):
        xt = torch.randn(tokens, hidden, device=DEV, generator=g).half()
        ins = {"x": xt, "freqs": f, "k_cache": c.k, "v_cache": c.v, "table": c.table, "lengths": c.lengths, "prefix_table": c.prefix_table}
        if ragged:
            ins["offsets"] = offsets
        kept = c.k.clone(), c.v.clone()
        out = torch.empty(tokens, hidden, device=DEV, dtype=torch.float16)
        module.run_with_tensors(ins, [out])
        written = c.k.clone(), c.v.clone()
        # the same through the eager calls, bit for bit
        c.k.copy_(kept[0]), c.v.copy_(kept[1])

        def eager_linear(t, name):
            tq, ts = eager.quantize_rows(t)
            return eager.gemm_rcr_int8(tq, w[name + "_w"], ts, w[name + "_s"], w[name + "_b"])

        rows = eager_linear(xt, "qkv").view(tokens, H + 2 * C, D)
        et = eager.paged_kv_append(rows[:, H:H + C], rows[:, H + C:], c.k, c.v, c.table, c.lengths, offsets, q=rows[:, :H], freqs=f,
                                   first_position=prefix)
        ey = eager.prefix_attention(et, c.k, c.v, c.table, c.lengths, offsets, prefix_table=c.prefix_table, prefix_length=prefix)
        want = eager_linear(ey.reshape(tokens, H * D), "out")
        assert torch.equal(c.k, written[0]) and torch.equal(c.v, written[1])
        assert torch.equal(out, want)
        # and next to plain torch, in 64 bits on the quantized operands
        plain(xt, w, f, kept, c, past if step == 0 else [p + n for p, n in zip(past, new)], new, starts, H, C, D, prefix, out)
        c.lengths += torch.tensor(new, dtype=torch.int32, device=DEV)


def plain(x, w, f, cache, c, past, new, starts, H, C, D, prefix, got):
    """The block in 64 bits.  Rounding to 8 bits decides differently next to a border, so the comparison is of the size of a step of
    the rows' quantization: 1 / 127 of the largest of a row of 512 numbers, summed with weights of 512 ** -0.5 (their norm is 1), is
    at most 2 / 127 of it."""
    from test_rotary_gpu import turned

    def linear(t, name):
        scale = t.abs().amax(1, keepdim=True) / 127.0
        q = (t / scale).round()
        return (q @ w[name + "_w"].double().t()) * scale * w[name + "_s"].double() + w[name + "_b"].double()

    rows = linear(x.double(), "qkv").half().view(-1, H + 2 * C, D)
    k_cache, v_cache = cache
    out = torch.empty(x.shape[0], H * D, dtype=torch.float64, device=DEV)
    for i, (p, n) in enumerate(zip(past, new)):
        mine = slice(starts[i], starts[i + 1])
        places = torch.arange(p, p + n, device=DEV)
        q, _ = turned(rows[mine, :H], places + prefix, f, False)
        k, _ = turned(rows[mine, H:H + C], places + prefix, f, False)
        k = torch.cat((c.read(k_cache, c.prefix_table, prefix).double(), c.read(k_cache, c.table[i], p).double(), k.half().double()))
        v = torch.cat((c.read(v_cache, c.prefix_table, prefix), c.read(v_cache, c.table[i], p), rows[mine, H + C:])).double()
        k, v = (t.repeat_interleave(H // C, 1).transpose(0, 1).contiguous() for t in (k, v))
        score = q.half().double().transpose(0, 1) @ k.transpose(1, 2).contiguous() * D ** -0.5
        hidden = torch.arange(prefix + p + n, device=DEV) >= prefix + torch.arange(p + 1, p + n + 1, device=DEV)[:, None]
        out[mine] = (torch.softmax(score.masked_fill(hidden, -torch.inf), -1) @ v).transpose(0, 1).reshape(n, H * D)
    want = linear(out.half().double(), "out")
    assert (got.double() - want).abs().max() <= out.abs().max() * 2 / 127 + want.abs().max() * 2.0 ** -9
