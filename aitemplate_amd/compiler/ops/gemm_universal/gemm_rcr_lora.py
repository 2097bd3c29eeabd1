"""gemm_rcr_lora: a projection that many requests share, with the low-rank adapter of each row's request (no counterpart in the
reference).

    y = ops.gemm_rcr_lora()(x, w, lora_a, lora_b, adapters, scales, bias)

y[m] = x[m] w^T (+ bias) + scales[i] (x[m] lora_a[i]^T) lora_b[i]^T with i = adapters[m], rounded once; rows whose number is not in
[0, adapters) have none."""
from typing import Optional

from ....backend import registry
from ....backend.target import Target
from ...base import IntImm, Operator, Tensor


class gemm_rcr_lora(Operator):
    def __init__(self) -> None:
        super().__init__()
        self._attrs["op"] = "gemm_rcr_lora"
        self._attrs["has_profiler"] = False

    def __call__(self, x: Tensor, w: Tensor, lora_a: Tensor, lora_b: Tensor, adapters: Tensor, scales: Optional[Tensor] = None,
                 bias: Optional[Tensor] = None) -> Tensor:
        from .... import _kernels

        dtype = x._attrs["dtype"]
        if dtype not in ("float16", "bfloat16"):
            raise RuntimeError(f"gemm_rcr_lora: x must be float16 or bfloat16, got {dtype}")
        for t, want, name in ((w, dtype, "w"), (lora_a, dtype, "lora_a"), (lora_b, dtype, "lora_b"), (adapters, "int32", "adapters"),
                              (scales, "float32", "scales"), (bias, dtype, "bias")):
            if t is not None and t._attrs["dtype"] != want:
                raise RuntimeError(f"gemm_rcr_lora: {name} must be {want}, got {t._attrs['dtype']}")
        shape, w_shape, a_shape, b_shape = (t._attrs["shape"] for t in (x, w, lora_a, lora_b))
        if len(shape) < 2 or len(w_shape) != 2 or shape[-1] != w_shape[1]:
            raise RuntimeError(f"A/B shape mismatch! A: {shape}, B: {w_shape}")
        if not isinstance(w_shape[0], IntImm) or not isinstance(w_shape[1], IntImm):
            raise RuntimeError("gemm_rcr_lora: N and K must be static")
        if len(a_shape) != 3 or a_shape[2] != w_shape[1] or not isinstance(a_shape[1], IntImm) or not 1 <= a_shape[1].value() <= 1024:
            raise RuntimeError("gemm_rcr_lora: lora_a must be [adapters, rank, K] with a static rank of 1 to 1024")
        if list(b_shape) != [a_shape[0], w_shape[0], a_shape[1]]:
            raise RuntimeError("gemm_rcr_lora: lora_b must be [adapters, N, rank]")
        if list(adapters._attrs["shape"]) != list(shape[:-1]):
            raise RuntimeError("gemm_rcr_lora: adapters must have one number for each row of x")
        for t, want, name in ((scales, a_shape[0], "scales [adapters]"), (bias, w_shape[0], "bias [N]")):
            if t is not None and list(t._attrs["shape"]) != [want]:
                raise RuntimeError(f"gemm_rcr_lora: {name} has shape {t._attrs['shape']}")
        self._attrs["inputs"] = [x, w, lora_a, lora_b, adapters] + [t for t in (scales, bias) if t is not None]
        self._attrs["has_scales"], self._attrs["has_bias"] = scales is not None, bias is not None
        self._set_depth()
        rows = 1
        for d in shape[:-1]:
            rows *= max(d._attrs["values"])
        # (fewer rows may want more: the library looks at what it gets)
        self._attrs["workspace"] = int(_kernels.load().aitamd_gemm_lora_workspace_bytes(
            _kernels.DTYPE_ID[dtype], -1, int(bias is not None), rows, w_shape[0].value(), w_shape[1].value(), a_shape[1].value()))
        output = Tensor(list(shape[:-1]) + [w_shape[0]], src_ops={self}, dtype=dtype)
        self._attrs["outputs"] = [output]
        return output

    def _get_op_attributes(self):
        return {}

    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)
