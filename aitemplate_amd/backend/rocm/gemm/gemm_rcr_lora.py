"""Registry hooks of gemm_rcr_lora: one generated function, the rows (the product of the leading dims, which may be dynamic) and the
number of adapters as its arguments, N, K and the rank as literals."""
from typing import Any, Dict

from ... import registry
from . import common


def _signature(func_name: str) -> str:
    return (f"void {func_name}(void* out, const void* x, const void* w, const void* lora_a, const void* lora_b, const void* adapters, "
            "const void* scales, const void* bias, uint8_t* workspace, int64_t workspace_bytes, int64_t rows, int64_t num_adapters, "
            "hipStream_t stream)")


def gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name, x = func_attrs["name"], func_attrs["inputs"][0]
    dtype = common.DTYPE_ID[x._attrs["dtype"]]
    n, k = (d.value() for d in func_attrs["inputs"][1]._attrs["shape"])
    rank = func_attrs["inputs"][2]._attrs["shape"][1].value()
    # (the instance table of products with adapters: see aitamd_gemm_rcr_lora)
    return f"""{common.header_with_table(int(func_attrs["has_bias"]), 4 + dtype)}
{_signature(func_name)} {{
  if (rows == 0) return;  // empty output
  check_rc(aitamd_gemm_rcr_lora({dtype}, -1, x, w, bias, lora_a, lora_b, static_cast<const int32_t*>(adapters),
                                static_cast<const float*>(scales), out, rows, {n}, {k}, {rank}, num_adapters, {k}, {k}, {n}, workspace,
                                workspace_bytes, stream), "{func_name}");
}}
{common.FOOTER}"""


def func_decl(func_attrs: Dict[str, Any]) -> str:
    return _signature(func_attrs["name"]) + ";"


def func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    inputs = [t._attrs["name"] for t in func_attrs["inputs"]]
    rest = inputs[5:]
    scales = rest.pop(0) if func_attrs["has_scales"] else "nullptr"
    bias = rest.pop(0) if func_attrs["has_bias"] else "nullptr"
    rows = " * ".join(d._attrs["name"] for d in func_attrs["inputs"][0]._attrs["shape"][:-1]) or "1"
    args = [func_attrs["outputs"][0]._attrs["name"]] + inputs[:5] + [scales, bias, "workspace_", "workspace_size_", rows,
                                                                     func_attrs["inputs"][2]._attrs["shape"][0]._attrs["name"], "stream"]
    return f"{indent}{func_attrs['name']}({', '.join(args)});"


registry.reg("rocm.gemm_rcr_lora.gen_function", gen_function)
registry.reg("rocm.gemm_rcr_lora.func_decl", func_decl)
registry.reg("rocm.gemm_rcr_lora.func_call", func_call)
