"""Registry hooks of rotary_embedding, qk_norm_rotary, paged_kv_append and prefix_attention: one generated function each, heads, head dims and the
page size as literals, the numbers of tokens, sequences and pages (which may be dynamic) as its arguments."""
from typing import Any, Dict

from ... import registry
from ..elementwise.elementwise import float_literal
from ..gemm import common


def _name(t) -> str:
    return t._attrs["name"]


def _dim(t, i: int) -> str:
    return t._attrs["shape"][i]._attrs["name"]


def _value(t, i: int) -> int:
    return t._attrs["shape"][i].value()


# ---- rotary_embedding ----

def _rotary_signature(func_name: str) -> str:
    return (f"void {func_name}(void* out, const void* x, const void* positions, const void* freqs, int64_t batch, int64_t seq, "
            "hipStream_t stream)")


def rotary_gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name = func_attrs["name"]
    x, positions, freqs = func_attrs["inputs"]
    heads, head_dim = _value(x, -2), _value(x, -1)
    row = heads * head_dim
    strides = f"seq * {row}, {row}, {head_dim}"
    return f"""{common.HEADER}
{_rotary_signature(func_name)} {{
  check_rc(aitamd_rotary_embedding({common.DTYPE_ID[x._attrs["dtype"]]}, x, out, positions, {int(positions._attrs["dtype"] == "int64")},
                                   static_cast<const float*>(freqs), batch, seq, {heads}, {head_dim}, {2 * _value(freqs, 0)}, {strides},
                                   {strides}, {"seq" if len(positions._attrs["shape"]) == 2 else "0"}, 1,
                                   {float_literal(func_attrs["scale"])}, {int(func_attrs["interleaved"])}, {int(func_attrs["inverse"])},
                                   stream), "{func_name}");
}}
{common.FOOTER}"""


def rotary_func_decl(func_attrs: Dict[str, Any]) -> str:
    return _rotary_signature(func_attrs["name"]) + ";"


def rotary_func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    x = func_attrs["inputs"][0]
    batch = _dim(x, 0) if len(x._attrs["shape"]) == 4 else "1"
    args = [_name(func_attrs["outputs"][0])] + [_name(t) for t in func_attrs["inputs"]] + [batch, _dim(x, -3), "stream"]
    return f"{indent}{func_attrs['name']}({', '.join(args)});"


# ---- qk_norm_rotary ----

def _norm_signature(func_name: str) -> str:
    return (f"void {func_name}(void* q_out, void* k_out, const void* q, const void* k, const void* q_weight, const void* k_weight, "
            "const void* positions, const void* freqs, int64_t batch, int64_t seq, hipStream_t stream)")


def norm_gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name = func_attrs["name"]
    q, k, q_weight, k_weight, positions, freqs = func_attrs["inputs"]
    head_dim = _value(q, -1)

    def heads(name, x, weight):
        strides = f"seq * {_value(x, -2) * head_dim}, {_value(x, -2) * head_dim}, {head_dim}"
        return (f"  const aitamd_heads {name}_heads = {{{name}, {name}_out, {_value(x, -2)}, {strides}, {strides}, {name}_weight, "
                f"{_weight_stride(weight)}}};")

    return f"""{common.HEADER}
{_norm_signature(func_name)} {{
{heads("q", q, q_weight)}
{heads("k", k, k_weight)}
  check_rc(aitamd_qk_norm_rotary({common.DTYPE_ID[q._attrs["dtype"]]}, &q_heads, &k_heads, positions,
                                 {int(positions._attrs["dtype"] == "int64")}, static_cast<const float*>(freqs), batch, seq, {head_dim},
                                 {2 * _value(freqs, 0)}, {"seq" if len(positions._attrs["shape"]) == 2 else "0"}, 1,
                                 {float_literal(func_attrs["eps"])}, {float_literal(func_attrs["scale"])},
                                 {int(func_attrs["interleaved"])}, stream), "{func_name}");
}}
{common.FOOTER}"""


def norm_func_decl(func_attrs: Dict[str, Any]) -> str:
    return _norm_signature(func_attrs["name"]) + ";"


def norm_func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    q = func_attrs["inputs"][0]
    batch = _dim(q, 0) if len(q._attrs["shape"]) == 4 else "1"
    args = [_name(t) for t in func_attrs["outputs"] + func_attrs["inputs"]] + [batch, _dim(q, -3), "stream"]
    return f"{indent}{func_attrs['name']}({', '.join(args)});"


# ---- the paged cache ----

_CACHE_PARAMS = ("void* k_cache, void* v_cache, const void* block_table, const void* lengths, const void* offsets, int64_t ends, "
                 "int64_t tokens, int64_t batch, int64_t pages, int64_t max_pages")


def _cache_code(func_name: str, k_cache) -> str:
    """The cache's description; `ends`: the number of offsets, which the kernels follow to offsets[batch]."""
    page_size, kv_heads, head_dim = (_value(k_cache, i) for i in (1, 2, 3))
    strides = f"{page_size * kv_heads * head_dim}, {kv_heads * head_dim}, {head_dim}"
    return (f'  if (offsets != nullptr && ends != batch + 1)\n    throw std::runtime_error("{func_name}: " + std::to_string(ends) + '
            '" offsets for " + std::to_string(batch) + " sequences (batch + 1 are wanted)");\n'
            f"  const aitamd_paged_cache cache = {{k_cache, v_cache, pages, {page_size}, {kv_heads}, {head_dim}, {strides},\n"
            f"                                    {strides}, static_cast<const int32_t*>(block_table), max_pages, max_pages,\n"
            "                                    static_cast<const int32_t*>(lengths), static_cast<const int32_t*>(offsets), batch, tokens};")


def _cache_args(q, k_cache, v_cache, block_table, lengths, offsets):
    ends = [_name(offsets), _dim(offsets, 0)] if offsets is not None else ["nullptr", "0"]
    return [_name(k_cache), _name(v_cache), _name(block_table), _name(lengths)] + ends + [
            _dim(q, 0), _dim(lengths, 0), _dim(k_cache, 0), _dim(block_table, 1)]


def _append_signature(func_name: str) -> str:
    return (f"void {func_name}(void* out, const void* q, const void* k, const void* v, const void* freqs, {_CACHE_PARAMS}, "
            "const void* q_weight, const void* k_weight, hipStream_t stream)")


def _append_options(func_attrs: Dict[str, Any]) -> Dict[str, Any]:
    """The optional inputs that there are, by name."""
    return dict(zip(func_attrs["optional_inputs"], func_attrs["inputs"][8:]))


def _weight_stride(weight) -> int:
    """From one head's weights to the next's."""
    return _value(weight, 1) if weight is not None and len(weight._attrs["shape"]) == 2 else 0


def append_gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name = func_attrs["name"]
    q, _, _, k_cache, _, _, _, freqs = func_attrs["inputs"][:8]
    heads, head_dim, kv_heads = _value(q, 1), _value(q, 2), _value(k_cache, 2)
    options = _append_options(func_attrs)
    q_weight, k_weight = options.get("q_weight"), options.get("k_weight")
    entry, norms = "aitamd_paged_kv_append", ""
    if q_weight is not None or k_weight is not None:
        entry += "_norm"
        norms = f"q_weight, {_weight_stride(q_weight)}, k_weight, {_weight_stride(k_weight)}, {float_literal(func_attrs['eps'])}, "
    return f"""{common.HEADER}
{_append_signature(func_name)} {{
{_cache_code(func_name, k_cache)}
  check_rc({entry}({common.DTYPE_ID[q._attrs["dtype"]]}, &cache, k, {kv_heads * head_dim}, {head_dim}, v,
                                  {kv_heads * head_dim}, {head_dim}, q, {heads * head_dim}, {head_dim}, out, {heads * head_dim},
                                  {head_dim}, {heads}, {norms}static_cast<const float*>(freqs), {2 * _value(freqs, 0)},
                                  {func_attrs["first_position"]}, {float_literal(func_attrs["scale"])},
                                  {int(func_attrs["interleaved"])}, stream), "{func_name}");
}}
{common.FOOTER}"""


def append_func_decl(func_attrs: Dict[str, Any]) -> str:
    return _append_signature(func_attrs["name"]) + ";"


def append_func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    q, k, v, k_cache, v_cache, block_table, lengths, freqs = func_attrs["inputs"][:8]
    options = _append_options(func_attrs)
    args = [_name(func_attrs["outputs"][0])] + [_name(t) for t in (q, k, v, freqs)]
    args += _cache_args(q, k_cache, v_cache, block_table, lengths, options.get("offsets"))
    args += [_name(options[w]) if w in options else "nullptr" for w in ("q_weight", "k_weight")] + ["stream"]
    return f"{indent}{func_attrs['name']}({', '.join(args)});"


def _attention_signature(func_name: str) -> str:
    return (f"void {func_name}(void* out, const void* q, {_CACHE_PARAMS}, const void* prefix_table, int64_t prefix_pages, "
            "uint8_t* workspace, int64_t workspace_bytes, hipStream_t stream)")


def attention_gen_function(func_attrs: Dict[str, Any]) -> str:
    func_name = func_attrs["name"]
    q, k_cache = func_attrs["inputs"][:2]
    heads, head_dim = _value(q, 1), _value(q, 2)
    scale = head_dim ** -0.5 if func_attrs["scale"] is None else func_attrs["scale"]
    # (behind the first 4096 bytes of the shared workspace, which other ops keep zero)
    return f"""{common.HEADER}
{_attention_signature(func_name)} {{
{_cache_code(func_name, k_cache)}
  check_rc(aitamd_prefix_attention({common.DTYPE_ID[q._attrs["dtype"]]}, &cache, q, {heads * head_dim}, {head_dim}, out,
                                   {heads * head_dim}, {head_dim}, {heads}, static_cast<const int32_t*>(prefix_table), prefix_pages,
                                   {func_attrs["prefix_length"]}, {float_literal(scale)}, workspace + 4096, workspace_bytes - 4096,
                                   stream), "{func_name}");
}}
{common.FOOTER}"""


def attention_func_decl(func_attrs: Dict[str, Any]) -> str:
    return _attention_signature(func_attrs["name"]) + ";"


def attention_func_call(func_attrs: Dict[str, Any], indent: str = "  ") -> str:
    q, k_cache, v_cache, block_table, lengths = func_attrs["inputs"][:5]
    rest = list(func_attrs["inputs"][5:])
    offsets = rest.pop(0) if func_attrs["has_offsets"] else None
    prefix = rest.pop(0) if rest else None
    args = [_name(func_attrs["outputs"][0]), _name(q)] + _cache_args(q, k_cache, v_cache, block_table, lengths, offsets)
    args += [_name(prefix), _dim(prefix, 0)] if prefix is not None else ["nullptr", "0"]
    return f"{indent}{func_attrs['name']}({', '.join(args + ['workspace_', 'workspace_size_', 'stream'])});"


registry.reg("rocm.rotary_embedding.gen_function", rotary_gen_function)
registry.reg("rocm.rotary_embedding.func_decl", rotary_func_decl)
registry.reg("rocm.rotary_embedding.func_call", rotary_func_call)
registry.reg("rocm.qk_norm_rotary.gen_function", norm_gen_function)
registry.reg("rocm.qk_norm_rotary.func_decl", norm_func_decl)
registry.reg("rocm.qk_norm_rotary.func_call", norm_func_call)
registry.reg("rocm.paged_kv_append.gen_function", append_gen_function)
registry.reg("rocm.paged_kv_append.func_decl", append_func_decl)
registry.reg("rocm.paged_kv_append.func_call", append_func_call)
registry.reg("rocm.prefix_attention.gen_function", attention_gen_function)
registry.reg("rocm.prefix_attention.func_decl", attention_func_decl)
registry.reg("rocm.prefix_attention.func_call", attention_func_call)
