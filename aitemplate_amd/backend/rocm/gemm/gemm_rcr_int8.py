"""Registry hooks of quantize_rows and gemm_rcr_int8: one generated function each, the rows (the product of the leading dims, which
may be dynamic) as its argument and K and N as literals."""
from typing import Any, Dict

from ... import registry
from . import common


def _rows(t) -> str:
    return " * ".join(d._attrs["name"] for d in t._attrs["shape"][:-1]) or "1"


def _quantize_signature(func_name: str) -> str:
    return f"void {func_name}(void* out, void* scale, const void* x, int64_t rows, hipStream_t stream)"


def quantize_gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name, x = func_attrs["name"], func_attrs["inputs"][0]
    columns = x._attrs["shape"][-1].value()
    return f"""{common.HEADER}
{_quantize_signature(func_name)} {{
  check_rc(aitamd_quantize_rows({common.DTYPE_ID[x._attrs["dtype"]]}, x, static_cast<int8_t*>(out), static_cast<float*>(scale), rows,
                                {columns}, {columns}, {columns}, stream), "{func_name}");
}}
{common.FOOTER}"""


def quantize_func_decl(func_attrs: Dict[str, Any]) -> str:
    return _quantize_signature(func_attrs["name"]) + ";"


def quantize_func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    x = func_attrs["inputs"][0]
    args = [t._attrs["name"] for t in func_attrs["outputs"]] + [x._attrs["name"], _rows(x), "stream"]
    return f"{indent}{func_attrs['name']}({', '.join(args)});"


def _gemm_signature(func_name: str) -> str:
    return (f"void {func_name}(void* out, const void* a, const void* b, const void* a_scale, const void* b_scale, const void* bias, "
            "uint8_t* workspace, int64_t workspace_bytes, int64_t rows, hipStream_t stream)")


def gemm_gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name = func_attrs["name"]
    dtype = common.DTYPE_ID[func_attrs["dtype"]]
    n, k = (d.value() for d in func_attrs["inputs"][1]._attrs["shape"])
    # (the instance table of 8-bit operands: see aitamd_gemm_rcr_int8)
    return f"""{common.header_with_table(1 if len(func_attrs["inputs"]) > 4 else 0, 2 + dtype)}
{_gemm_signature(func_name)} {{
  if (rows == 0) return;  // empty output
  check_rc(aitamd_gemm_rcr_int8({dtype}, -1, static_cast<const int8_t*>(a), static_cast<const int8_t*>(b),
                                static_cast<const float*>(a_scale), static_cast<const float*>(b_scale), bias, out, rows, {n}, {k}, {k},
                                {k}, {n}, workspace, workspace_bytes, stream), "{func_name}");
}}
{common.FOOTER}"""


def gemm_func_decl(func_attrs: Dict[str, Any]) -> str:
    return _gemm_signature(func_attrs["name"]) + ";"


def gemm_func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    inputs = [t._attrs["name"] for t in func_attrs["inputs"]]
    ws = ["workspace_", "workspace_size_"] if common.uses_workspace(func_attrs) else ["nullptr", "0"]
    args = [func_attrs["outputs"][0]._attrs["name"]] + inputs[:4] + (inputs[4:] or ["nullptr"]) + ws
    return f"{indent}{func_attrs['name']}({', '.join(args + [_rows(func_attrs['inputs'][0]), 'stream'])});"


registry.reg("rocm.quantize_rows.gen_function", quantize_gen_function)
registry.reg("rocm.quantize_rows.func_decl", quantize_func_decl)
registry.reg("rocm.quantize_rows.func_call", quantize_func_call)
registry.reg("rocm.gemm_rcr_int8.gen_function", gemm_gen_function)
registry.reg("rocm.gemm_rcr_int8.func_decl", gemm_func_decl)
registry.reg("rocm.gemm_rcr_int8.func_call", gemm_func_call)
