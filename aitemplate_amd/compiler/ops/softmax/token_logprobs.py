"""token_logprobs: log probabilities and ranks of given tokens, entropies and the most probable tokens of rows of logits, in one pass
(no counterpart in the reference).

    logprob, entropy, rank, top_logprob, top_token = ops.token_logprobs(top=8)(logits, tokens)

Of softmax(scale * logits) over the last dimension; see `eager.token_logprobs` for rows without numbers and tokens out of range."""
from typing import Tuple

from ....backend import registry
from ....backend.target import Target
from ...base import IntImm, Operator, Tensor

MOST_TOP = 64


class token_logprobs(Operator):
    def __init__(self, top: int = 0, scale: float = 1.0) -> None:
        super().__init__()
        self._attrs["op"] = "token_logprobs"
        self._attrs["has_profiler"] = False
        self._attrs["top"] = int(top)
        self._attrs["scale"] = float(scale)
        if not 0 <= self._attrs["top"] <= MOST_TOP:
            raise RuntimeError(f"token_logprobs: top {top}: 0 to {MOST_TOP}")
        if not 0.0 < self._attrs["scale"] < 2e38:  # (its product with log2(e) is a number of 32 bits too)
            raise RuntimeError(f"token_logprobs: scale {scale} is no positive number")

    def __call__(self, logits: Tensor, tokens: Tensor) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
        top = self._attrs["top"]
        if logits._attrs["dtype"] not in ("float16", "bfloat16", "float32"):
            raise RuntimeError(f"token_logprobs: logits must be float16, bfloat16 or float32, got {logits._attrs['dtype']}")
        if tokens._attrs["dtype"] not in ("int32", "int64"):
            raise RuntimeError(f"token_logprobs: tokens must be int32 or int64, got {tokens._attrs['dtype']}")
        shape = logits._attrs["shape"]
        if len(shape) < 2 or not isinstance(shape[-1], IntImm) or not max(top, 1) <= shape[-1].value():
            raise RuntimeError("token_logprobs: logits must be [..., vocabulary] with a static vocabulary of at least `top` tokens")
        if list(tokens._attrs["shape"]) != list(shape[:-1]):
            raise RuntimeError("token_logprobs: tokens must have one number for each row of logits")
        self._attrs["inputs"] = [logits, tokens]
        self._set_depth()
        # Parts of rows have workgroups of their own only where the rows leave CUs idle: all together at most two a CU, of 256 of them
        # (the library checks what it gets).  Behind the first 4096 bytes of the model's workspace, which the GEMMs that share
        # tiles keep zero.
        self._attrs["workspace"] = 4096 + 2 * 256 * ((16 + 8 * top + 15) // 16 * 16)
        lead = list(shape[:-1])
        self._attrs["outputs"] = ([Tensor(lead, src_ops={self}, dtype=d) for d in ("float32", "float32", "int32")]
                                  + ([Tensor(lead + [IntImm(top)], src_ops={self}, dtype=d) for d in ("float32", "int32")] if top else []))
        return tuple(self._attrs["outputs"])

    def _get_op_attributes(self):
        return {name: self._attrs[name] for name in ("top", "scale")}

    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)
