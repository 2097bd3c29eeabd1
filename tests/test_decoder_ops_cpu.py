"""The decoder operators as graph ops, without a GPU: shapes, hooks, refusals."""
import pytest

from aitemplate_amd.backend import registry
from aitemplate_amd.compiler import ops
from aitemplate_amd.compiler.dtype import dtype_enum_value, dtype_to_enumerator, get_dtype_size
from aitemplate_amd.frontend import IntImm, IntVar, Tensor
from aitemplate_amd.testing import detect_target


def tensor(name, shape, dtype="float16"):
    return Tensor(shape=[d if isinstance(d, IntVar) else IntImm(d) for d in shape], dtype=dtype, name=name, is_input=True)


def generated(op, name):
    from aitemplate_amd.backend import rocm  # noqa: F401

    from aitemplate_amd.compiler.transform.name_graph import name_graph
    from aitemplate_amd.compiler.transform.toposort import toposort

    op._attrs["outputs"][0]._attrs["is_output"] = True
    with detect_target():
        name_graph(toposort(op._attrs["outputs"][0]))
        op._attrs["name"] = name
        kind = op._attrs["op"]
        return (op.gen_function(), registry.get(f"rocm.{kind}.func_decl")(op._attrs), registry.get(f"rocm.{kind}.func_call")(op._attrs))


def test_int8_is_a_type_of_the_graph():
    assert get_dtype_size("int8") == 1 and dtype_enum_value("int8") == 7 and dtype_to_enumerator("int8") == "AITemplateDtype::kInt8"


def test_quantized_linear():
    m = IntVar(values=[1, 64], name="m")
    x = tensor("x", [m, 256])
    q_op, g_op = ops.quantize_rows(), ops.gemm_rcr_int8("bfloat16")
    q, scale = q_op(x)
    assert q._attrs["dtype"] == "int8" and scale._attrs["dtype"] == "float32"
    assert q._attrs["shape"] == x._attrs["shape"] and scale._attrs["shape"] == x._attrs["shape"][:-1]
    w, ws, b = tensor("w", [96, 256], "int8"), tensor("ws", [96], "float32"), tensor("b", [96], "bfloat16")
    y = g_op(q, w, scale, ws, b)
    assert y._attrs["dtype"] == "bfloat16" and y._attrs["shape"] == [m, IntImm(96)]
    source, decl, call = generated(g_op, "linear")
    assert "aitamd_gemm_rcr_int8(1, -1" in source and "aitamd_gemm_table_1_3" in source and decl.endswith(";") and "linear(" in call
    source, _, call = generated(q_op, "rows")
    assert "aitamd_quantize_rows(0, " in source and call.strip().startswith("rows(")
    other = tensor("other", [m, 128], "int8")
    for bad in (lambda: ops.quantize_rows()(tensor("i", [4, 8], "float32")), lambda: ops.quantize_rows()(tensor("i", [8])),
                lambda: ops.gemm_rcr_int8("float32"), lambda: ops.gemm_rcr_int8()(x, w, scale, ws),
                lambda: ops.gemm_rcr_int8()(other, w, scale, ws), lambda: ops.gemm_rcr_int8()(q, w, ws, ws),
                lambda: ops.gemm_rcr_int8()(q, w, scale, ws, b)):
        with pytest.raises(RuntimeError):
            bad()


def test_rotary():
    s = IntVar(values=[1, 64], name="s")
    x, positions, freqs = tensor("x", [2, s, 4, 64]), tensor("p", [s], "int32"), tensor("f", [16], "float32")
    op = ops.rotary_embedding(interleaved=True, scale=1.25)
    y = op(x, positions, freqs)
    assert y._attrs["shape"] == x._attrs["shape"] and y._attrs["dtype"] == "float16"
    source, _, call = generated(op, "turn")
    assert "aitamd_rotary_embedding(0, x, out, positions, 0," in source and "1.25f, 1, 0," in source and "turn(" in call
    for bad in ((tensor("x", [s, 64]), positions, freqs), (x, tensor("p", [3], "int32"), freqs), (x, positions, tensor("f", [33], "float32")),
                (x, positions, tensor("f", [16])), (x, tensor("p", [s], "float32"), freqs)):
        with pytest.raises(RuntimeError):
            ops.rotary_embedding()(*bad)


def cache(page=16, heads=2, dim=64, dtype="float16"):
    pages = IntVar(values=[1, 100], name="pages")
    return [tensor(n, [pages, page, heads, dim], dtype) for n in ("k_cache", "v_cache")]


def test_paged_cache():
    t, b = IntVar(values=[1, 64], name="t"), IntVar(values=[1, 8], name="b")
    q, k, v = tensor("q", [t, 8, 64]), tensor("k", [t, 2, 64]), tensor("v", [t, 2, 64])
    table, lengths = tensor("table", [b, IntVar(values=[1, 9], name="w")], "int32"), tensor("lengths", [b], "int32")
    offsets, freqs, prefix = tensor("offsets", [IntVar(values=[2, 9], name="e")], "int32"), tensor("f", [32], "float32"), tensor("shared", [5], "int32")
    append, attend = ops.paged_kv_append(first_position=70), ops.prefix_attention(prefix_length=70)
    y = append(q, k, v, *cache(), table, lengths, freqs, offsets)
    z = attend(y, *append._attrs["inputs"][3:5], table, lengths, offsets, prefix)
    assert y._attrs["shape"] == z._attrs["shape"] == q._attrs["shape"]
    assert attend._attrs["workspace"] >= 4096 + 2 * 64 * 8 * (64 * 4 + 8)
    source, _, call = generated(attend, "look")
    assert "aitamd_prefix_attention(0, &cache" in source and "workspace + 4096" in source and "shared, " in call and "offsets" in call
    source, _, call = generated(append, "put")
    assert "aitamd_paged_kv_append(0, &cache" in source and "70, 1.0f," in source and "offsets" in call
    one = [tensor("q", [b, 8, 64]), *cache(), table, lengths]
    ops.prefix_attention()(*one)
    for bad in (lambda: ops.prefix_attention()(q, *cache(), table, lengths),                      # rows without offsets
                lambda: ops.prefix_attention()(*one, prefix_table=prefix),                        # a prefix without a length
                lambda: ops.prefix_attention(5)(*one),
                lambda: ops.prefix_attention()(one[0], *cache(page=24), table, lengths),
                lambda: ops.prefix_attention()(one[0], *cache(heads=3), table, lengths),
                lambda: ops.prefix_attention()(one[0], *cache(dtype="bfloat16"), table, lengths),
                lambda: ops.paged_kv_append()(q, k, tensor("v", [t, 1, 64]), *cache(), table, lengths, freqs, offsets),
                lambda: ops.paged_kv_append()(q, k, v, y, y, table, lengths, freqs, offsets),
                lambda: ops.paged_kv_append()(q, k, v, *cache(), table, lengths, tensor("f", [33], "float32"), offsets)):
        with pytest.raises(RuntimeError):
            bad()
