"""rotary_embedding: positions turned into the heads of [..., heads, head_dim] operands (no counterpart in the reference).

The first 2 len(freqs) dims of every head: dims i and len(freqs) + i, or with `interleaved` 2 i and 2 i + 1, become
scale * (x1 cos - x2 sin, x2 cos + x1 sin) of the angle position * freqs[i]; `inverse` turns back (the gradient)."""
from ....backend import registry
from ....backend.target import Target
from ...base import IntImm, Operator, Tensor


def static_dim(t: Tensor, dim: int, what: str) -> int:
    """The value of a dim that the kernels take as a constant."""
    d = t._attrs["shape"][dim]
    if not isinstance(d, IntImm):
        raise RuntimeError(f"{what} must be static")
    return d.value()


def check_dtypes(op: str, **wanted) -> None:
    """`wanted`: name = (tensor or None, allowed dtypes)."""
    for name, (t, dtypes) in wanted.items():
        if t is not None and t._attrs["dtype"] not in dtypes:
            raise RuntimeError(f"{op}: {name} must be {' or '.join(dtypes)}, got {t._attrs['dtype']}")


def check_freqs(op: str, freqs: Tensor, head_dim: int) -> int:
    """The number of rotated dims."""
    if len(freqs._attrs["shape"]) != 1 or 2 * static_dim(freqs, 0, f"{op}: the number of frequencies") > head_dim:
        raise RuntimeError(f"{op}: freqs must be [n] with 2 n <= head_dim = {head_dim}")
    return 2 * static_dim(freqs, 0, "")


class rotary_embedding(Operator):
    def __init__(self, interleaved: bool = False, scale: float = 1.0, inverse: bool = False) -> None:
        super().__init__()
        self._attrs["op"] = "rotary_embedding"
        self._attrs["has_profiler"] = False
        self._attrs["interleaved"] = bool(interleaved)
        self._attrs["scale"] = float(scale)
        self._attrs["inverse"] = bool(inverse)

    def __call__(self, x: Tensor, positions: Tensor, freqs: Tensor) -> Tensor:
        shape, places = x._attrs["shape"], positions._attrs["shape"]
        if len(shape) not in (3, 4):
            raise RuntimeError("rotary_embedding: x must be [tokens, heads, head_dim] or [batch, seq, heads, head_dim]")
        check_dtypes("rotary_embedding", x=(x, ("float16", "bfloat16")), positions=(positions, ("int32", "int64")),
                     freqs=(freqs, ("float32",)))
        if list(places) not in (list(shape[:-2]), list(shape[-3:-2])):
            raise RuntimeError("rotary_embedding: positions must be [tokens], [batch, seq] or [seq]")
        static_dim(x, -2, "rotary_embedding: the number of heads")
        check_freqs("rotary_embedding", freqs, static_dim(x, -1, "rotary_embedding: head_dim"))
        self._attrs["inputs"] = [x, positions, freqs]
        self._set_depth()
        output = Tensor(list(shape), src_ops={self}, dtype=x._attrs["dtype"])
        self._attrs["outputs"] = [output]
        return output

    def _get_op_attributes(self):
        return {name: self._attrs[name] for name in ("interleaved", "scale", "inverse")}

    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)
