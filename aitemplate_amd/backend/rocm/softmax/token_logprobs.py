"""Registry hooks of token_logprobs: one generated function, the rows (the product of the leading dims, which may be dynamic) as its
argument, the vocabulary as a literal."""
from typing import Any, Dict

from ... import registry
from ..elementwise.elementwise import float_literal
from ..gemm import common

_DTYPE_ID = {"float16": 0, "bfloat16": 1, "float32": 8}


def _signature(func_name: str) -> str:
    return (f"void {func_name}(void* logprob, void* entropy, void* rank, void* top_logprob, void* top_token, const void* logits, "
            "const void* tokens, uint8_t* workspace, int64_t workspace_bytes, int64_t rows, hipStream_t stream)")


def gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name = func_attrs["name"]
    logits, tokens = func_attrs["inputs"]
    vocabulary = logits._attrs["shape"][-1].value()
    # (behind the first 4096 bytes of the shared workspace, which other ops keep zero)
    return f"""{common.HEADER}
{_signature(func_name)} {{
  check_rc(aitamd_token_logprobs({_DTYPE_ID[logits._attrs["dtype"]]}, logits, tokens, {int(tokens._attrs["dtype"] == "int64")},
                                 static_cast<float*>(logprob), static_cast<float*>(entropy), static_cast<int32_t*>(rank),
                                 static_cast<float*>(top_logprob), static_cast<int32_t*>(top_token), rows, {vocabulary}, {vocabulary},
                                 {func_attrs["top"]}, {float_literal(func_attrs["scale"])}, workspace + 4096, workspace_bytes - 4096,
                                 stream), "{func_name}");
}}
{common.FOOTER}"""


def func_decl(func_attrs: Dict[str, Any]) -> str:
    return _signature(func_attrs["name"]) + ";"


def func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    logits, tokens = func_attrs["inputs"]
    outs = [t._attrs["name"] for t in func_attrs["outputs"]]
    rows = " * ".join(d._attrs["name"] for d in logits._attrs["shape"][:-1])
    args = outs + ["nullptr"] * (5 - len(outs)) + [logits._attrs["name"], tokens._attrs["name"], "workspace_", "workspace_size_", rows, "stream"]
    return f"{indent}{func_attrs['name']}({', '.join(args)});"


registry.reg("rocm.token_logprobs.gen_function", gen_function)
registry.reg("rocm.token_logprobs.func_decl", func_decl)
registry.reg("rocm.token_logprobs.func_call", func_call)
