"""paged_kv_append and prefix_attention: a step's keys and values into a cache of pages, and the attention of its rows over it
(no counterpart in the reference).

The cache is a pair of model inputs [pages, page_size, kv_heads, head_dim], which `paged_kv_append` writes in place.  Its
result, the rotated queries, is what `prefix_attention` takes: so the one runs behind the other.  `block_table` [batch, n],
`lengths` [batch] (tokens that the sequences have in their pages before the step) and `offsets` [batch + 1] (the sequences' rows;
without it row i is sequence i's) are int32 inputs."""
from typing import Optional

from ....backend import registry
from ....backend.target import Target
from ...base import Operator, Tensor
from .rotary_embedding import check_dtypes, check_freqs, static_dim


def _check_cache(op: str, q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, offsets: Optional[Tensor]):
    dtype = q._attrs["dtype"]
    check_dtypes(op, q=(q, ("float16", "bfloat16")), k_cache=(k_cache, (dtype,)), v_cache=(v_cache, (dtype,)),
                 block_table=(block_table, ("int32",)), lengths=(lengths, ("int32",)), offsets=(offsets, ("int32",)))
    if len(q._attrs["shape"]) != 3:
        raise RuntimeError(f"{op}: q must be [tokens, heads, head_dim]")
    if len(k_cache._attrs["shape"]) != 4 or list(k_cache._attrs["shape"]) != list(v_cache._attrs["shape"]):
        raise RuntimeError(f"{op}: k_cache and v_cache must be [pages, page_size, kv_heads, head_dim]")
    heads, head_dim = static_dim(q, 1, f"{op}: the number of heads"), static_dim(q, 2, f"{op}: head_dim")
    for dim, what in ((1, "page_size"), (2, "the number of key heads"), (3, "head_dim")):
        static_dim(k_cache, dim, f"{op}: {what}")
    if static_dim(k_cache, 3, "") != head_dim or heads % static_dim(k_cache, 2, ""):
        raise RuntimeError(f"{op}: the heads of q and of the cache do not match")
    if len(block_table._attrs["shape"]) != 2 or len(lengths._attrs["shape"]) != 1 or (offsets is not None and len(offsets._attrs["shape"]) != 1):
        raise RuntimeError(f"{op}: block_table must be [batch, pages of a sequence], lengths [batch], offsets [batch + 1]")
    if offsets is not None:
        # (numbers of their own in the graph: where they may fit, a run checks that they do)
        ends, batch = offsets._attrs["shape"][0]._attrs["values"], lengths._attrs["shape"][0]._attrs["values"]
        if max(ends) < min(batch) + 1 or min(ends) > max(batch) + 1:
            raise RuntimeError(f"{op}: offsets must be [batch + 1], got {ends} for batch {batch}")
    if block_table._attrs["shape"][0] != lengths._attrs["shape"][0]:
        raise RuntimeError(f"{op}: block_table and lengths differ in the number of sequences")
    if offsets is None and q._attrs["shape"][0] != lengths._attrs["shape"][0]:
        raise RuntimeError(f"{op}: without offsets every sequence has one row")
    return heads, head_dim


class _paged(Operator):
    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)

    def _finish(self, q: Tensor, inputs) -> Tensor:
        self._attrs["inputs"] = inputs
        self._set_depth()
        output = Tensor(list(q._attrs["shape"]), src_ops={self}, dtype=q._attrs["dtype"])
        self._attrs["outputs"] = [output]
        return output


class paged_kv_append(_paged):
    """Keys and values [tokens, kv_heads, head_dim] into the cache, keys and queries rotated on the way (as by `rotary_embedding`, for
    position first_position + the token's place in its sequence); returns the rotated queries."""

    def __init__(self, interleaved: bool = False, scale: float = 1.0, first_position: int = 0) -> None:
        super().__init__()
        self._attrs["op"] = "paged_kv_append"
        self._attrs["has_profiler"] = False
        self._attrs["interleaved"] = bool(interleaved)
        self._attrs["scale"] = float(scale)
        self._attrs["first_position"] = int(first_position)

    def __call__(self, q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor,
                 freqs: Tensor, offsets: Optional[Tensor] = None) -> Tensor:
        _, head_dim = _check_cache("paged_kv_append", q, k_cache, v_cache, block_table, lengths, offsets)
        for t, name in ((k, "k"), (v, "v")):
            check_dtypes("paged_kv_append", **{name: (t, (q._attrs["dtype"],))})
            if list(t._attrs["shape"]) != [q._attrs["shape"][0]] + list(k_cache._attrs["shape"][2:]):
                raise RuntimeError(f"paged_kv_append: {name} must be [tokens, kv_heads, head_dim]")
        for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            if not t._attrs["is_input"]:
                # (neither another op's result nor a constant, which the runtimes of a container share)
                raise RuntimeError(f"paged_kv_append: {name} is written in place and must be an input of the model")
        check_dtypes("paged_kv_append", freqs=(freqs, ("float32",)))
        if check_freqs("paged_kv_append", freqs, head_dim) == 0:
            raise RuntimeError("paged_kv_append: freqs is empty")
        return self._finish(q, [q, k, v, k_cache, v_cache, block_table, lengths, freqs] + ([] if offsets is None else [offsets]))

    def _get_op_attributes(self):
        return {name: self._attrs[name] for name in ("interleaved", "scale", "first_position")}


class prefix_attention(_paged):
    """Attention of the rows q over the first `prefix_length` keys of the pages in `prefix_table` [n], which all sequences share, and
    those of their own pages up to themselves; scale head_dim ** -0.5 unless given."""

    def __init__(self, prefix_length: int = 0, scale: Optional[float] = None) -> None:
        super().__init__()
        self._attrs["op"] = "prefix_attention"
        self._attrs["has_profiler"] = False
        self._attrs["prefix_length"] = int(prefix_length)
        self._attrs["scale"] = scale

    def __call__(self, q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor,
                 offsets: Optional[Tensor] = None, prefix_table: Optional[Tensor] = None) -> Tensor:
        heads, head_dim = _check_cache("prefix_attention", q, k_cache, v_cache, block_table, lengths, offsets)
        if head_dim % 8 or head_dim > 256 or static_dim(k_cache, 1, "") % 16:
            raise RuntimeError("prefix_attention: head_dim must be a multiple of 8 up to 256, page_size one of 16")
        if (self._attrs["prefix_length"] > 0) != (prefix_table is not None):
            raise RuntimeError("prefix_attention: prefix_table goes with a prefix_length above 0")
        if prefix_table is not None:
            check_dtypes("prefix_attention", prefix_table=(prefix_table, ("int32",)))
            if len(prefix_table._attrs["shape"]) != 1:
                raise RuntimeError("prefix_attention: prefix_table must be [pages of the prefix]")
        # Scratch memory: parts of a row's keys are taken by workgroups of their own only where the rows leave CUs idle, so the
        # parts of all rows are at most twice the rows, or twice the chip's (the library checks what it gets).  Behind the first
        # 4096 bytes of the model's workspace, which the GEMMs that share tiles keep zero.
        rows = max(q._attrs["shape"][0]._attrs["values"]) * heads
        self._attrs["workspace"] = 4096 + 2 * (rows + 2 * 256 * 128) * (head_dim * 4 + 8)
        self._attrs["has_offsets"] = offsets is not None
        return self._finish(q, [q, k_cache, v_cache, block_table, lengths] + [t for t in (offsets, prefix_table) if t is not None])

    def _get_op_attributes(self):
        return {name: self._attrs[name] for name in ("prefix_length", "scale")}
