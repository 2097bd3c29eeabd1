"""quantize_rows and gemm_rcr_int8: rows as 8-bit integers with a scale each, and the product of such rows with a weight of 8-bit
integers that has a scale for each output channel (no counterpart in the reference).

    x_q, x_scale = ops.quantize_rows()(x)
    y = ops.gemm_rcr_int8()(x_q, w_q, x_scale, w_scale, bias)

The sums are exact (32-bit integers); y = x_scale * w_scale * sum + bias, rounded once to fp16 or bf16."""
from typing import Optional, Tuple

from ....backend import registry
from ....backend.target import Target
from ...base import IntImm, Operator, Tensor


class quantize_rows(Operator):
    """Rows of x [..., K] as (int8 [..., K], float32 [...]): scale = max|x| / 127, whole numbers nearest to x / scale."""

    def __init__(self) -> None:
        super().__init__()
        self._attrs["op"] = "quantize_rows"
        self._attrs["has_profiler"] = False

    def __call__(self, x: Tensor) -> Tuple[Tensor, Tensor]:
        if x._attrs["dtype"] not in ("float16", "bfloat16"):
            raise RuntimeError(f"quantize_rows: x must be float16 or bfloat16, got {x._attrs['dtype']}")
        shape = x._attrs["shape"]
        if len(shape) < 2 or not isinstance(shape[-1], IntImm):
            raise RuntimeError("quantize_rows: x must be [..., K] with a static K")
        self._attrs["inputs"] = [x]
        self._set_depth()
        self._attrs["outputs"] = [Tensor(list(shape), src_ops={self}, dtype="int8"), Tensor(list(shape[:-1]), src_ops={self}, dtype="float32")]
        return tuple(self._attrs["outputs"])

    def _get_op_attributes(self):
        return {}

    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)


class gemm_rcr_int8(Operator):
    def __init__(self, dtype: str = "float16") -> None:
        super().__init__()
        if dtype not in ("float16", "bfloat16"):
            raise RuntimeError(f"gemm_rcr_int8: the result must be float16 or bfloat16, got {dtype}")
        self._attrs["op"] = "gemm_rcr_int8"
        self._attrs["has_profiler"] = False
        self._attrs["dtype"] = dtype

    def __call__(self, a: Tensor, b: Tensor, a_scale: Tensor, b_scale: Tensor, bias: Optional[Tensor] = None) -> Tensor:
        from .... import _kernels

        dtype = self._attrs["dtype"]
        for t, want, name in ((a, "int8", "a"), (b, "int8", "b"), (a_scale, "float32", "a_scale"), (b_scale, "float32", "b_scale"),
                              (bias, dtype, "bias")):
            if t is not None and t._attrs["dtype"] != want:
                raise RuntimeError(f"gemm_rcr_int8: {name} must be {want}, got {t._attrs['dtype']}")
        a_shape, b_shape = a._attrs["shape"], b._attrs["shape"]
        if len(a_shape) < 2 or len(b_shape) != 2 or a_shape[-1] != b_shape[1]:
            raise RuntimeError(f"A/B shape mismatch! A: {a_shape}, B: {b_shape}")
        if not isinstance(b_shape[0], IntImm) or not isinstance(b_shape[1], IntImm):
            raise RuntimeError("gemm_rcr_int8: N and K must be static")
        if list(a_scale._attrs["shape"]) != list(a_shape[:-1]):
            raise RuntimeError("gemm_rcr_int8: a_scale must have one number for each row of a")
        for t, name in ((b_scale, "b_scale"), (bias, "bias")):
            if t is not None and list(t._attrs["shape"]) != [b_shape[0]]:
                raise RuntimeError(f"gemm_rcr_int8: {name} must be [N]")
        self._attrs["inputs"] = [a, b, a_scale, b_scale] + ([] if bias is None else [bias])
        self._set_depth()
        rows = 1
        for d in a_shape[:-1]:
            rows *= max(d._attrs["values"])
        # (fewer rows may want more: the library looks at what it gets)
        self._attrs["workspace"] = int(_kernels.load().aitamd_gemm_int8_workspace_bytes(
            _kernels.DTYPE_ID[dtype], -1, int(bias is not None), rows, b_shape[0].value(), b_shape[1].value()))
        output = Tensor(list(a_shape[:-1]) + [b_shape[0]], src_ops={self}, dtype=dtype)
        self._attrs["outputs"] = [output]
        return output

    def _get_op_attributes(self):
        return {"dtype": self._attrs["dtype"]}

    def gen_function(self) -> str:
        return registry.get(f"{Target.current().name()}.{self._attrs['op']}.gen_function")(self._attrs)
