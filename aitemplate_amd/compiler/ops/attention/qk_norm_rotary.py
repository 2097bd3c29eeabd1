"""qk_norm_rotary: heads of queries and keys, normalized and rotated in one launch (no counterpart in the reference).

Every head x of q and k becomes x / sqrt(mean(x ** 2) + eps) * weight, with weights [head_dim] or [heads, head_dim], and is then
turned as by `rotary_embedding`."""
from typing import Tuple

from ....backend import registry
from ....backend.target import Target
from ...base import Operator, Tensor
from .rotary_embedding import check_dtypes, check_freqs, static_dim


def check_weight(op: str, name: str, weight: Tensor, x: Tensor) -> None:
    dims = [d.value() for d in x._attrs["shape"][-2:]]
    shape = [static_dim(weight, i, f"{op}: {name}") for i in range(len(weight._attrs["shape"]))]
    check_dtypes(op, **{name: (weight, (x._attrs["dtype"],))})
    if shape not in (dims[1:], dims):
        raise RuntimeError(f"{op}: {name} must be {dims[1:]} or {dims}, got {shape}")


def check_eps(op: str, eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise RuntimeError(f"{op}: eps {eps} is no number of at least 0")
    return eps


class qk_norm_rotary(Operator):
    def __init__(self, eps: float = 1e-6, interleaved: bool = False, scale: float = 1.0) -> None:
        super().__init__()
        self._attrs["op"] = "qk_norm_rotary"
        self._attrs["has_profiler"] = False
        self._attrs["eps"] = check_eps("qk_norm_rotary", eps)
        self._attrs["interleaved"] = bool(interleaved)
        self._attrs["scale"] = float(scale)

    def __call__(self, q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, positions: Tensor, freqs: Tensor) -> Tuple[Tensor, Tensor]:
        shape, k_shape, places = (t._attrs["shape"] for t in (q, k, positions))
        if len(shape) not in (3, 4):
            raise RuntimeError("qk_norm_rotary: q must be [tokens, heads, head_dim] or [batch, seq, heads, head_dim]")
        check_dtypes("qk_norm_rotary", q=(q, ("float16", "bfloat16")), k=(k, (q._attrs["dtype"],)), positions=(positions, ("int32", "int64")),
                     freqs=(freqs, ("float32",)))
        if len(k_shape) != len(shape) or list(k_shape[:-2]) != list(shape[:-2]) or k_shape[-1] != shape[-1]:
            raise RuntimeError(f"qk_norm_rotary: k of shape {k_shape} does not fit q of shape {shape}")
        if list(places) not in (list(shape[:-2]), list(shape[-3:-2])):
            raise RuntimeError("qk_norm_rotary: positions must be [tokens], [batch, seq] or [seq]")
        for t in (q, k):
            static_dim(t, -2, "qk_norm_rotary: the number of heads")
        check_freqs("qk_norm_rotary", freqs, static_dim(q, -1, "qk_norm_rotary: head_dim"))
        check_weight("qk_norm_rotary", "q_weight", q_weight, q)
        check_weight("qk_norm_rotary", "k_weight", k_weight, k)
        self._attrs["inputs"] = [q, k, q_weight, k_weight, positions, freqs]
        self._set_depth()
        self._attrs["outputs"] = [Tensor(list(t._attrs["shape"]), src_ops={self}, dtype=q._attrs["dtype"]) for t in (q, k)]
        return tuple(self._attrs["outputs"])

    def _get_op_attributes(self):
        return {name: self._attrs[name] for name in ("eps", "interleaved", "scale")}

    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)
