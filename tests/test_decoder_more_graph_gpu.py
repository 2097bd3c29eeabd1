"""Adapters beside a projection, normalized heads and log probabilities as graph ops against the eager calls (which have tests of
their own), through both paths of those, on another stream, and a step of a decoder that runs them together: eager, as a graph and
captured, against plain torch in 64 bits."""
import itertools
import os

import pytest
import torch

from aitemplate_amd import _kernels, eager
from aitemplate_amd.compiler import compile_model, ops
from aitemplate_amd.frontend import IntImm, IntVar, Tensor
from aitemplate_amd.testing import detect_target
from paged_common import DEV, Paged

pytestmark = pytest.mark.gpu

WORKDIR = os.environ.get("AIT_TEST_WORKDIR", "/tmp/aitemplate_amd_tests")
_counter = itertools.count()
TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def build(outputs):
    for i, t in enumerate(outputs):
        t._attrs["name"], t._attrs["is_output"] = f"output_{i}", True
    return compile_model(list(outputs), detect_target(), WORKDIR, f"more_{next(_counter)}")


def feed(name, shape, dtype):
    return Tensor(shape=[IntImm(d) if isinstance(d, int) else d for d in shape], dtype=dtype, name=name, is_input=True)


def normal(*shape, dtype=torch.float16, scale=1.0):
    return (torch.randn(*shape, device=DEV) * scale).to(dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("N,K,rank,bias,scales", [(96, 256, 8, True, True), (33, 130, 5, False, True), (520, 1024, 16, False, False), (64, 64, 40, True, False)])
def test_lora(dtype, N, K, rank, bias, scales):
    m, n = IntVar(values=[1, 300], name="m"), IntVar(values=[1, 9], name="n")
    t = [feed("x", [m, K], dtype), feed("w", [N, K], dtype), feed("a", [n, rank, K], dtype), feed("b", [n, N, rank], dtype), feed("of", [m], "int32"),
         feed("scales", [n], "float32") if scales else None, feed("bias", [N], dtype) if bias else None]
    module = build([ops.gemm_rcr_lora()(*t)])
    for rows, adapters in ((300, 9), (1, 1), (37, 5)):
        ins = {"x": normal(rows, K, dtype=TORCH[dtype]), "w": normal(N, K, dtype=TORCH[dtype], scale=K ** -0.5),
               "a": normal(adapters, rank, K, dtype=TORCH[dtype], scale=K ** -0.5), "b": normal(adapters, N, rank, dtype=TORCH[dtype]),
               "of": torch.randint(-1, adapters, (rows,), device=DEV, dtype=torch.int32), "scales": torch.rand(adapters, device=DEV) if scales else None,
               "bias": normal(N, dtype=TORCH[dtype]) if bias else None}
        out = torch.empty(rows, N, device=DEV, dtype=TORCH[dtype])
        module.run_with_tensors({k: v for k, v in ins.items() if v is not None}, [out])
        assert torch.equal(out, eager.gemm_rcr_lora(*ins.values()))


@pytest.mark.parametrize("dtype,interleaved", [("float16", False), ("bfloat16", True)])
def test_norm(dtype, interleaved):
    batch, seq = IntVar(values=[1, 4], name="batch"), IntVar(values=[1, 40], name="seq")
    q, k = feed("q", [batch, seq, 6, 64], dtype), feed("k", [batch, seq, 2, 64], dtype)
    qw, kw = feed("qw", [64], dtype), feed("kw", [2, 64], dtype)
    positions, freqs = feed("positions", [batch, seq], "int64"), feed("freqs", [16], "float32")
    module = build(list(ops.qk_norm_rotary(1e-5, interleaved, 1.5)(q, k, qw, kw, positions, freqs)))
    for b, s in ((4, 40), (1, 1)):
        ins = {"q": normal(b, s, 6, 64, dtype=TORCH[dtype]), "k": normal(b, s, 2, 64, dtype=TORCH[dtype]), "qw": normal(64, dtype=TORCH[dtype]),
               "kw": normal(2, 64, dtype=TORCH[dtype]), "positions": torch.randint(0, 10000, (b, s), device=DEV),
               "freqs": eager.rotary_frequencies(32, device=DEV)[0]}
        outs = [torch.empty_like(ins["q"]), torch.empty_like(ins["k"])]
        module.run_with_tensors(ins, outs)
        want = eager.qk_norm_rotary(*ins.values(), eps=1e-5, interleaved=interleaved, scale=1.5)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("dtype,token,top,scale", [("float16", "int64", 5, 0.7), ("bfloat16", "int32", 0, 1.0), ("float32", "int64", 64, 1.0)])
def test_logprobs(dtype, token, top, scale):
    m = IntVar(values=[1, 40], name="m")
    module = build(list(ops.token_logprobs(top=top, scale=scale)(feed("logits", [m, 9001], dtype), feed("tokens", [m], token))))
    for rows in (40, 1):
        logits = normal(rows, 9001, dtype=TORCH[dtype], scale=3.0)
        tokens = torch.randint(-1, 9001, (rows,), device=DEV).to(getattr(torch, token))
        outs = [torch.empty(rows, device=DEV), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV, dtype=torch.int32)]
        if top:
            outs += [torch.empty(rows, top, device=DEV), torch.empty(rows, top, device=DEV, dtype=torch.int32)]
        module.run_with_tensors({"logits": logits, "tokens": tokens}, outs)
        for got, want in zip(outs, eager.token_logprobs(logits, tokens, top, scale)):
            assert torch.equal(got, want)


class Step:
    """Rows of several requests: a projection to queries, keys and values with each request's adapter, norms and rotation into the
    cache, attention, a projection with adapters, and the log probabilities of given tokens under a head."""
    H, C, D, HIDDEN, PAGE, RANK, N, V, TOP, EPS = 8, 2, 64, 320, 16, 12, 5, 1000, 4, 1e-5

    def __init__(self, past, new, seed=0):
        torch.manual_seed(seed)
        self.past, self.new = past, new
        self.c = Paged(torch.float16, past, new, self.C, self.D, self.PAGE, ragged=True)
        self.c.k.nan_to_num_(0.0), self.c.v.nan_to_num_(0.0)
        self.tokens = self.c.tokens
        wide, flat = (self.H + 2 * self.C) * self.D, self.H * self.D
        self.w = {}
        for name, n, k in (("qkv", wide, self.HIDDEN), ("out", self.HIDDEN, flat)):
            self.w[name + "_w"], self.w[name + "_bias"] = normal(n, k, scale=k ** -0.5), normal(n, scale=0.1)
            self.w[name + "_a"], self.w[name + "_b"] = normal(self.N, self.RANK, k, scale=k ** -0.5), normal(self.N, n, self.RANK, scale=0.2)
        self.w["q_norm"], self.w["k_norm"] = normal(self.D) * 0.2 + 1, normal(self.C, self.D) * 0.2 + 1
        self.w["head"] = normal(self.V, self.HIDDEN, scale=0.1)
        self.scales = torch.rand(self.N, device=DEV) + 0.5
        self.freqs = eager.rotary_frequencies(self.D, device=DEV)[0]
        self.x = normal(self.tokens, self.HIDDEN)
        self.wanted = torch.randint(0, self.V, (self.tokens,), device=DEV)
        self.of = torch.randint(-1, self.N, (len(new),), device=DEV, dtype=torch.int32).repeat_interleave(torch.tensor(new, device=DEV))

    def eager(self):
        c, w, D = self.c, self.w, self.D
        rows = eager.gemm_rcr_lora(self.x, w["qkv_w"], w["qkv_a"], w["qkv_b"], self.of, self.scales, w["qkv_bias"]).view(self.tokens, -1, D)
        q, k, v = rows.split([self.H, self.C, self.C], 1)
        q = eager.paged_kv_append(k, v, c.k, c.v, c.table, c.lengths, c.offsets, q=q, freqs=self.freqs, q_weight=w["q_norm"], k_weight=w["k_norm"],
                                  eps=self.EPS)
        y = eager.prefix_attention(q, c.k, c.v, c.table, c.lengths, c.offsets).view(self.tokens, -1)
        y = eager.gemm_rcr_lora(y, w["out_w"], w["out_a"], w["out_b"], self.of, self.scales, w["out_bias"])
        logits = eager.gemm("gemm_rcr", y, w["head"])
        return (*eager.token_logprobs(logits, self.wanted, self.TOP), logits)

    def module(self):
        T, B = IntVar(values=[1, 64], name="tokens"), IntVar(values=[1, 8], name="sequences")
        P = IntVar(values=[1, 64], name="pages")
        x, of, wanted = feed("x", [T, self.HIDDEN], "float16"), feed("of", [T], "int32"), feed("wanted", [T], "int64")
        scales, freqs = feed("scales", [self.N], "float32"), feed("freqs", [self.D // 2], "float32")
        k_cache, v_cache = (feed(n, [P, self.PAGE, self.C, self.D], "float16") for n in ("k_cache", "v_cache"))
        table, lengths = feed("table", [B, IntVar(values=[1, 16], name="most")], "int32"), feed("lengths", [B], "int32")
        offsets = feed("offsets", [IntVar(values=[2, 9], name="ends")], "int32")

        def constant(name):
            return Tensor([IntImm(d) for d in self.w[name].shape], dtype="float16", name=name)

        def project(t, name):
            return ops.gemm_rcr_lora()(t, constant(name + "_w"), constant(name + "_a"), constant(name + "_b"), of, scales, constant(name + "_bias"))

        D, sizes = self.D, (self.H, self.C, self.C)
        parts = ops.split()(project(x, "qkv"), [n * D for n in sizes], 1)
        q, k, v = (ops.reshape()(t, [T, n, D]) for t, n in zip(parts, sizes))
        q = ops.paged_kv_append(eps=self.EPS)(q, k, v, k_cache, v_cache, table, lengths, freqs, offsets, q_weight=constant("q_norm"),
                                              k_weight=constant("k_norm"))
        y = ops.prefix_attention()(q, k_cache, v_cache, table, lengths, offsets)
        y = project(ops.reshape()(y, [T, self.H * D]), "out")
        logits = ops.gemm_rcr()(y, constant("head"))
        module = build([*ops.token_logprobs(top=self.TOP)(logits, wanted), logits])
        module.set_many_constants_with_tensors(self.w)
        return module

    def plain(self):
        """In 64 bits, from the cache as it is."""
        w, c, D = {n: t.double() for n, t in self.w.items()}, self.c, self.D

        def project(t, name):
            y = t @ w[name + "_w"].t() + w[name + "_bias"]
            for m, i in enumerate(self.of.tolist()):
                if i >= 0:
                    y[m] += self.scales[i].double() * (t[m] @ w[name + "_a"][i].t()) @ w[name + "_b"][i].t()
            return y

        def head(t, weight, positions):
            t = t * (t.square().mean(-1, keepdim=True) + self.EPS).rsqrt() * weight
            angle = positions.double()[:, None] * self.freqs.double()
            cos, sin = angle.cos()[:, None], angle.sin()[:, None]
            a, b = t[..., :D // 2], t[..., D // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        positions = torch.cat([torch.arange(p, p + n, device=DEV) for p, n in zip(self.past, self.new)])
        q, k, v = project(self.x.double(), "qkv").view(self.tokens, -1, D).split([self.H, self.C, self.C], 1)
        q, k = head(q, w["q_norm"], positions), head(k, w["k_norm"], positions)
        rows = []
        for i, (p, n) in enumerate(zip(self.past, self.new)):
            own = slice(c.starts[i], c.starts[i] + n)
            ks = torch.cat([c.read(c.k, c.table[i], p).double(), k[own]]).repeat_interleave(self.H // self.C, 1)
            vs = torch.cat([c.read(c.v, c.table[i], p).double(), v[own]]).repeat_interleave(self.H // self.C, 1)
            for j in range(n):
                m, seen = c.starts[i] + j, p + j + 1
                s = (ks[:seen] * q[m]).sum(-1) * D ** -0.5
                rows.append((s.softmax(0)[..., None] * vs[:seen]).sum(0).reshape(-1))
        logits = project(torch.stack(rows), "out") @ w["head"].t()
        log = logits.log_softmax(-1)
        return log.gather(1, self.wanted[:, None])[:, 0], -(log.exp() * log).sum(-1), logits

    def keep(self):
        return self.c.k.clone(), self.c.v.clone()

    def restore(self, kept):
        self.c.k.copy_(kept[0]), self.c.v.copy_(kept[1])


@pytest.mark.parametrize("past,new", [([20, 3, 40, 0], [1, 1, 1, 1]), ([20, 3, 0, 40], [5, 1, 9, 0]), ([0], [1])])
def test_together(past, new):
    step = Step(past, new)
    kept = step.keep()
    want, entropy, exact = step.plain()
    *got, logits = step.eager()
    # The plain form's logits have none of the roundings to a half on the way: rows of the projection, the heads, the attention,
    # the second projection and the logits themselves, each off by 2^-11 of numbers of the size of what they make up.  Each passes a
    # product of norm about one, so that the whole is off by some 5 x 2^-11 of the logits' size and its like at random; a wrong row,
    # adapter, norm or position is off by the size itself.
    size = exact.abs().max()
    assert (logits.double() - exact).abs().max() <= 16 * 2.0 ** -11 * size
    # ... and an error of e in every logit is one of 2 e at most in their log probabilities, and in the entropy of (largest distance + 1) times that
    assert (got[0].double() - want).abs().max() <= 2 * 16 * 2.0 ** -11 * size
    assert (got[1].double() - entropy).abs().max() <= 2 * 16 * 2.0 ** -11 * size * (2 * size + 1)
    for a, b in zip(got, eager.token_logprobs(logits, step.wanted, step.TOP)):
        assert torch.equal(a, b)
    written = step.keep()

    # as a graph
    step.restore(kept)
    outs = [torch.empty_like(t) for t in (*got, logits)]
    step.module().run_with_tensors({"x": step.x, "of": step.of, "wanted": step.wanted, "scales": step.scales, "freqs": step.freqs, "k_cache": step.c.k,
                                    "v_cache": step.c.v, "table": step.c.table, "lengths": step.c.lengths, "offsets": step.c.offsets}, outs)
    # (the head may be another instance of the plain product, which sums in another order: two roundings)
    assert (outs[-1].double() - logits.double()).abs().max() <= 2 * 2.0 ** -11 * size + 2.0 ** -20
    for a, b in zip(outs, eager.token_logprobs(outs[-1], step.wanted, step.TOP)):
        assert torch.equal(a, b)
    assert torch.equal(step.c.k, written[0]) and torch.equal(step.c.v, written[1])

    # captured, with other inputs at each replay and eager calls between
    step.restore(kept)
    step.eager()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step.eager()
    for _ in range(3):
        step.x.copy_(normal(*step.x.shape))
        step.of.copy_(torch.randint_like(step.of, -1, step.N))
        step.restore(kept)
        graph.replay()
        torch.cuda.synchronize()
        replayed, cache = [t.clone() for t in captured], step.keep()
        step.restore(kept)
        for a, b in zip(replayed, step.eager()):
            assert torch.equal(a, b)
        assert torch.equal(cache[0], step.c.k) and torch.equal(cache[1], step.c.v)


def test_two_graphs_in_turn_and_on_another_stream():
    """Two captured graphs and eager calls on a stream of their own, whose work the current stream has not waited for."""
    steps = [Step([20, 3, 40], [3, 1, 2], seed=1), Step([7], [1], seed=2)]
    want, graphs, outs = [], [], []
    for s in steps:
        want.append([t.clone() for t in s.eager()])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(s.eager())
    for order in ((0, 1), (1, 0, 0), (1, 1, 0)):
        for i in order:
            for t in outs[i]:
                t.zero_()
            graphs[i].replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            late = [torch.zeros_like(steps[0].x), torch.zeros_like(steps[1].x)]
            kept = [s.x for s in steps]
            for s, t in zip(steps, late):
                t.copy_(s.x)
                s.x = t
            got = [s.eager() for s in steps]
        side.synchronize()
        for s, x in zip(steps, kept):
            s.x = x
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def calls():
    g = torch.Generator(device=DEV).manual_seed(1)

    def some(*shape, dtype=torch.float16):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    x, w, a, b = some(6, 128), some(72, 128), some(3, 9, 128), some(3, 72, 9)
    of, scales, bias = torch.tensor([0, 2, -1, 1, 1, 3], dtype=torch.int32, device=DEV), torch.rand(3, device=DEV), some(72)
    q, k, v, qw, kw = some(6, 8, 64), some(6, 2, 64), some(6, 2, 64), some(64), some(2, 64)
    positions, freqs = torch.arange(6, device=DEV), eager.rotary_frequencies(64, device=DEV)[0]
    c = Paged(torch.float16, [20, 3, 40], [1, 3, 2], 2, 64, 16, 33)
    cache = (c.k, c.v, c.table, c.lengths, c.offsets)
    logits, tokens = some(6, 1000), torch.tensor([0, 999, -1, 5, 1000, 7], device=DEV)
    return {
        "lora": lambda: eager.gemm_rcr_lora(x, w, a, b, of),
        "lora_all": lambda: eager.gemm_rcr_lora(x, w, a, b, of, scales, bias),
        "lora_batches": lambda: eager.gemm_rcr_lora(x.view(2, 3, 128), w, a, b, of.view(2, 3), scales),
        "lora_out": lambda: eager.gemm_rcr_lora(x, w, a, b, of, bias=bias, out=torch.empty(6, 72, device=DEV).half()),
        "norm": lambda: eager.qk_norm_rotary(q, k, qw, kw, positions, freqs),
        "norm_batches": lambda: eager.qk_norm_rotary(q.view(2, 3, 8, 64), k.view(2, 3, 2, 64), qw, kw, positions[:3].int(), freqs, 1e-5, True, 0.5),
        "norm_alone": lambda: eager.qk_norm_rotary(q, None, qw, None, positions),
        "norm_out": lambda: eager.qk_norm_rotary(q, k, None, kw, positions, freqs, q_out=torch.empty_like(q), k_out=torch.empty_like(k)),
        "append": lambda: (eager.paged_kv_append(k, v, *cache, q=q, freqs=freqs, q_weight=qw, k_weight=kw), c.k.nan_to_num(0), c.v.nan_to_num(0)),
        "append_keys": lambda: (eager.paged_kv_append(k, v, *cache, freqs=freqs, k_weight=kw, eps=0.1), c.k.nan_to_num(0)),
        "append_queries": lambda: (eager.paged_kv_append(k, v, *cache, q=q, q_weight=qw, q_out=torch.empty_like(q)), c.k.nan_to_num(0)),
        "logprobs": lambda: eager.token_logprobs(logits, tokens),
        "logprobs_top": lambda: eager.token_logprobs(logits.view(2, 3, 1000), tokens.view(2, 3).int(), 7, 0.5),
        "logprobs_pitch": lambda: eager.token_logprobs(logits[:, :900].float(), tokens, 64),
    }


LEFT = ("lora_out", "norm_alone", "norm_out", "append_keys", "append_queries")  # calls that the module leaves to the Python path


@pytest.mark.parametrize("name", list(calls()) if torch.cuda.is_available() else [])
def test_both_paths(name, monkeypatch):
    call = calls()[name]
    leaves = lambda r: r if isinstance(r, tuple) else (r,)  # noqa: E731
    native = [t if t is None else t.clone() for t in leaves(call())]
    taken = []

    class Counted:
        def __getattr__(self, f):
            def run(*args):
                r = getattr(_kernels.load_native("_native_decoder"), f)(*args)
                taken.append(r is not NotImplemented)
                return r
            return run

    monkeypatch.setattr(eager, "_native_decoder", Counted())
    call()
    assert any(taken) == (name not in LEFT)
    monkeypatch.setattr(eager, "_native_decoder", _kernels._NoNative())
    for a, b in zip(native, leaves(call())):
        assert (a is None and b is None) or (a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K,rank", [(3, 64, 64, 8), (40, 136, 256, 12), (64, 1536, 2048, 16), (600, 512, 256, 40), (2100, 2048, 256, 16)])
@pytest.mark.parametrize("in_a", [False, True])
def test_an_adapter_that_is_no_numbers_is_its_own_requests_alone(dtype, M, N, K, rank, in_a):
    """Infinities and NaN in one adapter's halves: its rows have none that are numbers, and all others are the same to the bit as
    beside an adapter of zeros."""
    torch.manual_seed(M)
    x, w, b = normal(M, K, dtype=dtype), normal(N, K, dtype=dtype, scale=K ** -0.5), normal(N, dtype=dtype)
    la, lb = normal(6, rank, K, dtype=dtype, scale=K ** -0.5), normal(6, N, rank, dtype=dtype)
    for order in ("mixed", "in a row"):
        of = torch.randint(-1, 6, (M,), device=DEV, dtype=torch.int32)
        of[0], of[-1] = 2, 1
        if order == "in a row":
            of = of.sort()[0]
        bad_a, bad_b = la.clone(), lb.clone()
        (bad_a if in_a else bad_b)[2].fill_(float("inf"))
        (bad_a if in_a else bad_b)[2, 0].fill_(float("nan"))
        zero_a, zero_b = la.clone(), lb.clone()
        zero_a[2], zero_b[2] = 0, 0
        got, want = eager.gemm_rcr_lora(x, w, bad_a, bad_b, of, bias=b), eager.gemm_rcr_lora(x, w, zero_a, zero_b, of, bias=b)
        assert torch.equal(got[of != 2], want[of != 2]), order
        assert not torch.isfinite(got[of == 2]).any(), order
