"""Direct launches of the GEMM-family kernels on torch device tensors.

Each helper hands raw device pointers, sizes and the current HIP stream to the
C ABI of the kernel library (``include/aitemplate_amd_kernels.h``); torch is
used for memory and streams only.  The names and argument order follow the
reference frontend ops (``ops.gemm_rcr_bias()(a, b, bias)`` etc.,
python/aitemplate/compiler/ops/gemm_universal/).  There is no fallback path:
a missing library or a CPU tensor raises.

The calls with ordinary arguments (plain GPU tensors that fit, contiguous rows) go through the extension module
``_native`` (``csrc/native_calls.cpp``): the same checks and the same C ABI call, 2 to 3 us of host time instead of
12 to 16.  It returns NotImplemented for anything else, which the Python code here then handles or refuses; without
the module that code takes every call.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _kernels

_native = _kernels.load_native()
_native_decoder = _kernels.load_native("_native_decoder")

_TORCH_DTYPE_ID = {torch.float16: 0, torch.bfloat16: 1}


def _check(t: Optional[torch.Tensor], name: str, dtype=None):
    if t is None:
        return
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (no CPU path exists)")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype} differs from {dtype}")


def _stream_ptr() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t: Optional[torch.Tensor]) -> Optional[ctypes.c_void_p]:
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _row_pitch(t: torch.Tensor, name: str) -> int:
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be 2-D with a contiguous last dimension")
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], t.stride(0))


def gemm_workspace_bytes(op: str, algo: int, M: int, N: int, K: int, dtype=torch.float16, batch: int = 1) -> int:
    """Bytes of scratch memory instance `algo` of `op` needs for this problem (0 for all but the split-K ones)."""
    lib = _kernels.load()
    return int(lib.aitamd_gemm_workspace_bytes(_kernels.EPILOGUE_OF_OP[op], _TORCH_DTYPE_ID[dtype], algo, batch, M, N, K))


def new_workspace(nbytes: int, device="cuda") -> torch.Tensor:
    """A scratch buffer for `gemm(..., workspace=)`: zeroed once (the kernels leave its counters zero again)."""
    return torch.zeros(max(int(nbytes), 16), dtype=torch.uint8, device=device)


def gemm(op: str, a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None,
         d0: Optional[torch.Tensor] = None, d1: Optional[torch.Tensor] = None,
         out: Optional[torch.Tensor] = None, algo: int = -1,
         workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Run reference op `op` (e.g. "gemm_rcr_bias_gelu"): out = epilogue(a @ b.T, bias, d0, d1).

    `a` may have more than 2 dims; leading dims are flattened into M as the
    reference does (gemm_rcr.py:51-77).  `algo` = -1 uses the library heuristic,
    otherwise the instance index (see `_kernels.gemm_algo_names`).  `workspace`: a buffer from
    `new_workspace` for the instances that split K between workgroups (the reference ops' `workspace`
    attribute, gemm_common.py:201-215); without it those instances are not chosen.
    """
    result = _native.gemm(op, a, b, bias, d0, d1, out, algo, workspace)
    if result is not NotImplemented:
        return result
    lib = _kernels.load()
    epi = _kernels.EPILOGUE_OF_OP[op]
    dtype = a.dtype
    if dtype not in _TORCH_DTYPE_ID:
        raise ValueError(f"unsupported dtype {dtype}")
    for t, n in ((a, "a"), (b, "b"), (bias, "bias"), (d0, "d0"), (d1, "d1"), (out, "out")):
        _check(t, n, dtype)
    lead = a.shape[:-1]
    K = a.shape[-1]
    M = 1
    for d in lead:
        M *= d
    a2 = a.reshape(M, K)
    N = b.shape[0]
    if b.dim() != 2 or b.shape[1] != K:
        raise ValueError(f"b must be [N, K={K}], got {tuple(b.shape)}")
    if out is None:
        out = torch.empty(*lead, N, dtype=dtype, device=a.device)
    if out.dim() == 2 and out.shape == (M, N) and out.stride(1) == 1 and out.stride(0) >= N:
        out2 = out  # a row-pitched view (rows of a wider buffer) is written in place with ldc = its pitch
    else:
        _check_out(out, M * N, "M*N")
        out2 = out.view(M, N)
    nres = _kernels.NUM_RESIDUALS_OF_EPILOGUE[epi]
    if epi != 0 and (bias is None or bias.numel() != N or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous 1-D tensor of size N")
    d0_2 = d0.reshape(M, N) if d0 is not None else None
    d1_2 = d1.reshape(M, N) if d1 is not None else None
    if nres >= 1 and (d0_2 is None or d0_2.shape != out2.shape):
        raise ValueError("d0 must have the output's shape")
    if nres >= 2 and (d1_2 is None or d1_2.shape != out2.shape):
        raise ValueError("d1 must have the output's shape")
    ldd = _row_pitch(d0_2, "d0") if nres >= 1 else N
    if nres >= 2 and _row_pitch(d1_2, "d1") != ldd:
        raise ValueError("d0 and d1 must share a row pitch")
    if workspace is not None and (not workspace.is_cuda or not workspace.is_contiguous()
                                  or workspace.dtype != torch.uint8):
        raise ValueError("workspace must be a contiguous uint8 GPU tensor (see new_workspace)")
    rc = lib.aitamd_gemm_rcr_ws(epi, _TORCH_DTYPE_ID[dtype], algo, _p(a2), _p(b), _p(bias), _p(d0_2), _p(d1_2),
                                _p(out2), M, N, K, _row_pitch(a2, "a"), _row_pitch(b, "b"), _row_pitch(out2, "out"),
                                ldd, _p(workspace), 0 if workspace is None else workspace.numel(), _stream_ptr())
    _kernels.check(rc, op)
    return out


def _check_out(out: torch.Tensor, numel: int, what: str) -> None:
    """A caller's output buffer is written in place through its raw pointer: it has to be dense and of the
    result's size, or the kernel would write past it (or into a temporary copy)."""
    if not out.is_contiguous() or out.numel() != numel:
        raise ValueError(f"out must be contiguous with {what} = {numel} elements, got shape {tuple(out.shape)} "
                         f"strides {tuple(out.stride())}")


def gemm_permute(op: str, a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor], shape,
                 out: Optional[torch.Tensor] = None, algo: int = -1) -> torch.Tensor:
    """Run a permuting op (`_kernels.PERMUTE_OPS`): linear(a, b, bias) written through the op's 5-D permutation.

    `shape` = (t1, t2, t3) as in the reference ops (gemm_rcr_bias_permute.py:28-76, gemm_rcr_permute.py:33-70).
    Returns [t2, M/t1, t3, t1, N/(t2*t3)] for the m2n3 ops and [t2, M/(t1*t2), t3, t1, N/t3] for the others.
    """
    lib = _kernels.load()
    epi, layout = _kernels.PERMUTE_OPS[op]
    dtype = a.dtype
    if dtype not in _TORCH_DTYPE_ID:
        raise ValueError(f"unsupported dtype {dtype}")
    for t, n in ((a, "a"), (b, "b"), (bias, "bias"), (out, "out")):
        _check(t, n, dtype)
    operands = _kernels.LAYOUT_ID[_kernels.PERMUTE_OPERANDS.get(op, "rcr")]
    K = a.shape[-1]
    a2 = a.reshape(-1, K)
    b_k, b_n = (0, 1) if operands & 1 else (1, 0)  # gemm_rrr_bias_permute takes B as [K, N]
    if b.dim() != 2 or b.shape[b_k] != K:
        raise ValueError(f"b does not match K={K}: got {tuple(b.shape)}")
    M, N = a2.shape[0], b.shape[b_n]
    if epi != 0 and (bias is None or bias.numel() != N or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous 1-D tensor of size N")
    t1, t2, t3 = (int(t) for t in shape)
    if layout == _kernels.PERMUTE_M2N3:
        if M % t1 or N % (t2 * t3):
            raise ValueError(f"[{M}, {N}] does not split by shape {tuple(shape)}")
        out_shape = (t2, M // t1, t3, t1, N // (t2 * t3))
    else:
        if M % (t1 * t2) or N % t3:
            raise ValueError(f"[{M}, {N}] does not split by shape {tuple(shape)}")
        out_shape = (t2, M // (t1 * t2), t3, t1, N // t3)
    if out is None:
        out = torch.empty(out_shape, dtype=dtype, device=a.device)
    elif not out.is_contiguous() or out.numel() != M * N:
        raise ValueError("out must be contiguous with M*N elements")
    rc = lib.aitamd_gemm_permute(operands, epi, _TORCH_DTYPE_ID[dtype], algo, _p(a2), _p(b), _p(bias), _p(out), M, N, K,
                                 _row_pitch(a2, "a"), _row_pitch(b, "b"), layout, t1, t2, t3, _stream_ptr())
    _kernels.check(rc, op)
    return out


def bmm_rcr(a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None, algo: int = -1) -> torch.Tensor:
    """out[b] = a[b] @ b[b].T with batch broadcast when one operand is 2-D or has batch 1
    (python/aitemplate/compiler/ops/gemm_universal/bmm.py:72-90)."""
    result = _native.bmm(0, a, b, out, 0, algo, "bmm_rcr")
    if result is not NotImplemented:
        return result
    lib = _kernels.load()
    dtype = a.dtype
    for t, n in ((a, "a"), (b, "b"), (out, "out")):
        _check(t, n, dtype)
    a3 = a if a.dim() == 3 else a.unsqueeze(0)
    b3 = b if b.dim() == 3 else b.unsqueeze(0)
    if not (a3.is_contiguous() and b3.is_contiguous()):
        raise ValueError("bmm_rcr operands must be contiguous")
    B = max(a3.shape[0], b3.shape[0])
    if a3.shape[0] not in (1, B) or b3.shape[0] not in (1, B):
        raise ValueError("batch sizes must match or be 1")
    M, K = a3.shape[1], a3.shape[2]
    N = b3.shape[1]
    if b3.shape[2] != K:
        raise ValueError("K mismatch")
    if out is None:
        out = torch.empty(B, M, N, dtype=dtype, device=a.device)
    else:
        _check_out(out, B * M * N, "B*M*N")
    sa = 0 if (a3.shape[0] == 1 and B > 1) else M * K
    sb = 0 if (b3.shape[0] == 1 and B > 1) else N * K
    rc = lib.aitamd_bmm_rcr(_TORCH_DTYPE_ID[dtype], algo, _p(a3), _p(b3), _p(out), B, M, N, K, K, K, N, sa, sb,
                            M * N, _stream_ptr())
    _kernels.check(rc, "bmm_rcr")
    return out


def bmm(layout: str, a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None, d1: int = 0,
        algo: int = -1) -> torch.Tensor:
    """Batched GEMM for the operand layouts "rcr", "rrr", "ccr", "crr" of the reference
    (python/aitemplate/compiler/ops/gemm_universal/bmm_xxx.py): first letter r = A is [B, M, K], c = A is
    [B, K, M]; second letter r = B is [B, K, N], c = B is [B, N, K]; the result is [B, M, N], or
    [B // d1, M, d1, N] when d1 > 0 (the *_permute ops).  2-D or batch-1 operands broadcast."""
    lay = _kernels.LAYOUT_ID[layout]
    result = _native.bmm(lay, a, b, out, d1, algo, "bmm_" + layout)
    if result is not NotImplemented:
        return result
    lib = _kernels.load()
    dtype = a.dtype
    for t, n in ((a, "a"), (b, "b"), (out, "out")):
        _check(t, n, dtype)
    a3 = a if a.dim() == 3 else a.unsqueeze(0)
    b3 = b if b.dim() == 3 else b.unsqueeze(0)
    if not (a3.is_contiguous() and b3.is_contiguous()):
        raise ValueError("bmm operands must be contiguous")
    B = max(a3.shape[0], b3.shape[0])
    if a3.shape[0] not in (1, B) or b3.shape[0] not in (1, B):
        raise ValueError("batch sizes must match or be 1")
    M, K = (a3.shape[2], a3.shape[1]) if lay & 2 else (a3.shape[1], a3.shape[2])
    N, Kb = (b3.shape[2], b3.shape[1]) if lay & 1 else (b3.shape[1], b3.shape[2])
    if Kb != K:
        raise ValueError("K mismatch")
    if d1 and (d1 < 0 or B % d1):
        raise ValueError(f"batch {B} is not a multiple of d1 = {d1}")
    if out is None:
        out = torch.empty((B // d1, M, d1, N) if d1 else (B, M, N), dtype=dtype, device=a.device)
    elif not out.is_contiguous() or out.numel() != B * M * N:
        raise ValueError("out must be contiguous with B*M*N elements")
    sa = 0 if (a3.shape[0] == 1 and B > 1) else M * K
    sb = 0 if (b3.shape[0] == 1 and B > 1) else N * K
    rc = lib.aitamd_bmm(lay, _TORCH_DTYPE_ID[dtype], algo, _p(a3), _p(b3), _p(out), B, M, N, K, a3.shape[2],
                        b3.shape[2], N, sa, sb, M * N, d1, _stream_ptr())
    _kernels.check(rc, f"bmm_{layout}")
    return out


def bmm_add(layout: str, a: torch.Tensor, b: torch.Tensor, d0: torch.Tensor, out: Optional[torch.Tensor] = None,
            algo: int = -1) -> torch.Tensor:
    """bmm(layout, a, b) + d0 with d0 of the result's shape [B, M, N]: the bmm_rrr_add / bmm_ccr_add / bmm_crr_add
    ops (python/aitemplate/compiler/ops/gemm_universal/bmm_xxx_add.py)."""
    lib = _kernels.load()
    lay = _kernels.LAYOUT_ID[layout]
    dtype = a.dtype
    for t, n in ((a, "a"), (b, "b"), (d0, "d0"), (out, "out")):
        _check(t, n, dtype)
    if a.dim() != 3 or b.dim() != 3 or not (a.is_contiguous() and b.is_contiguous() and d0.is_contiguous()):
        raise ValueError("bmm_add operands must be contiguous 3-D tensors")
    B = a.shape[0]
    M, K = (a.shape[2], a.shape[1]) if lay & 2 else (a.shape[1], a.shape[2])
    N, Kb = (b.shape[2], b.shape[1]) if lay & 1 else (b.shape[1], b.shape[2])
    if Kb != K or b.shape[0] != B:
        raise ValueError("A and B do not match")
    if tuple(d0.shape) != (B, M, N):
        raise ValueError(f"d0 must be [{B}, {M}, {N}], got {tuple(d0.shape)}")
    if out is None:
        out = torch.empty(B, M, N, dtype=dtype, device=a.device)
    else:
        _check_out(out, B * M * N, "B*M*N")
    rc = lib.aitamd_bmm_add(lay, _TORCH_DTYPE_ID[dtype], algo, _p(a), _p(b), _p(d0), _p(out), B, M, N, K, a.shape[2],
                            b.shape[2], N, N, M * K, N * K, M * N, M * N, _stream_ptr())
    _kernels.check(rc, f"bmm_{layout}_add")
    return out


def bmm_rcr_permute(a: torch.Tensor, b: torch.Tensor, shape, out: Optional[torch.Tensor] = None,
                    algo: int = -1) -> torch.Tensor:
    """bmm_rcr stored as [B // d1, M, d1, N] with shape = (d1,)
    (python/aitemplate/compiler/ops/gemm_universal/bmm_rcr_permute.py:28-116)."""
    lib = _kernels.load()
    dtype = a.dtype
    for t, n in ((a, "a"), (b, "b"), (out, "out")):
        _check(t, n, dtype)
    a3 = a if a.dim() == 3 else a.unsqueeze(0)
    b3 = b if b.dim() == 3 else b.unsqueeze(0)
    if not (a3.is_contiguous() and b3.is_contiguous()):
        raise ValueError("bmm_rcr_permute operands must be contiguous")
    B = max(a3.shape[0], b3.shape[0])
    if a3.shape[0] not in (1, B) or b3.shape[0] not in (1, B):
        raise ValueError("batch sizes must match or be 1")
    M, K = a3.shape[1], a3.shape[2]
    N = b3.shape[1]
    if b3.shape[2] != K:
        raise ValueError("K mismatch")
    d1 = int(shape[0])
    if d1 <= 0 or B % d1:
        raise ValueError(f"batch {B} is not a multiple of d1 = {d1}")
    if out is None:
        out = torch.empty(B // d1, M, d1, N, dtype=dtype, device=a.device)
    elif not out.is_contiguous() or out.numel() != B * M * N:
        raise ValueError("out must be contiguous with B*M*N elements")
    sa = 0 if (a3.shape[0] == 1 and B > 1) else M * K
    sb = 0 if (b3.shape[0] == 1 and B > 1) else N * K
    rc = lib.aitamd_bmm_rcr_permute(_TORCH_DTYPE_ID[dtype], algo, _p(a3), _p(b3), _p(out), B, M, N, K, K, K, sa, sb,
                                    d1, _stream_ptr())
    _kernels.check(rc, "bmm_rcr_permute")
    return out


def bmm_softmax_bmm_permute(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, shape, scale: float = 1.0,
                            causal: bool = False, layout: str = "0213",
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q @ k^T) @ v with the [B, M, O] result written as [B / G, M, G, O], G = shape[0]
    (python/aitemplate/compiler/ops/gemm_universal/bmm_softmax_bmm_permute.py:30-194)."""
    if layout != "0213":
        raise NotImplementedError(f"{layout} is not implemented!")
    result = _native.bmm_softmax_bmm_permute(q, k, v, int(shape[0]), float(scale), bool(causal), out)
    if result is not NotImplemented:
        return result
    lib = _kernels.load()
    dtype = q.dtype
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        _check(t, n, dtype)
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        raise ValueError("bmm_softmax_bmm_permute operands must be contiguous")
    B, M, K = q.shape
    N, O = v.shape[1], v.shape[2]
    if k.shape != (B, N, K) or v.shape[0] != B:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}")
    G = int(shape[0])
    if out is None:
        out = torch.empty(B // G, M, G, O, dtype=dtype, device=q.device)
    else:
        _check_out(out, B * M * O, "B*M*O")
    rc = lib.aitamd_bmm_softmax_bmm_permute(_TORCH_DTYPE_ID[dtype], _p(q), _p(k), _p(v), _p(out), B, M, N, K, O, G,
                                            float(scale), int(bool(causal)), _stream_ptr())
    _kernels.check(rc, "bmm_softmax_bmm_permute")
    return out


def mem_eff_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False,
                      lengths_kv: Optional[torch.Tensor] = None, lengths_q: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q k^T / sqrt(head_dim)) v on [batch, heads, seq, head_dim] operands, written as
    [batch, seq_q, heads, head_dim_v]; `lengths_kv` ([batch] or [batch, 1], int32, on the device) limits batch entry b
    to its first lengths_kv[b] keys; `lengths_q`, same form, zeroes the query rows past lengths_q[b]
    (python/aitemplate/compiler/ops/attention/mem_eff_attention.py:49-263)."""
    result = _native.mem_eff_attention(q, k, v, bool(causal), lengths_kv, lengths_q, out)
    if result is not NotImplemented:
        return result
    lib = _kernels.load()
    dtype = q.dtype
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        _check(t, n, dtype)
    if not (q.dim() == k.dim() == v.dim() == 4):
        raise ValueError("mem_eff_attention operands must be [batch, heads, seq, head_dim]")
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        raise ValueError("mem_eff_attention operands must be contiguous")
    batch, heads, seq_q, head_dim = q.shape
    seq_kv, head_dim_v = v.shape[2], v.shape[3]
    if k.shape != (batch, heads, seq_kv, head_dim) or v.shape[:2] != (batch, heads):
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}")
    for lengths, name in ((lengths_kv, "lengths_kv"), (lengths_q, "lengths_q")):
        if lengths is not None and (lengths.dtype != torch.int32 or lengths.numel() != batch
                                    or not lengths.is_contiguous() or lengths.device != q.device):
            raise ValueError(f"{name} must be a contiguous int32 tensor with one entry per batch on the operands' device")
    if out is None:
        out = torch.empty(batch, seq_q, heads, head_dim_v, dtype=dtype, device=q.device)
    else:
        _check_out(out, batch * seq_q * heads * head_dim_v, "batch*seq_q*heads*head_dim_v")
    rc = lib.aitamd_mem_eff_attention(_TORCH_DTYPE_ID[dtype], _p(q), _p(k), _p(v), _p(out), batch, heads, seq_q, seq_kv,
                                      head_dim, head_dim_v, float(head_dim) ** -0.5, int(bool(causal)),
                                      _p(lengths_kv), _p(lengths_q), _stream_ptr())
    _kernels.check(rc, "mem_eff_attention")
    return out


def elementwise(func: str, a: torch.Tensor, b=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stand-alone element-wise op `func` (a FuncEnum name, e.g. "ADD", "FASTGELU"): f(a, b) with b a tensor whose
    shape is a's or a suffix of it (leading 1s allowed), a number, or None for the unary functions.  A number or a
    broadcast tensor as the FIRST operand: pass it as `a` and the full-shape tensor as `b`."""
    from .compiler.ops.common.epilogue import FuncEnum

    lib = _kernels.load()
    fid = FuncEnum[func].value
    swap = 0
    if not isinstance(a, torch.Tensor) or (isinstance(b, torch.Tensor) and b.numel() > a.numel()):
        a, b, swap = b, a, 1
    _check(a, "a", None)
    if a.dtype not in _TORCH_DTYPE_ID or not a.is_contiguous():
        raise ValueError("a must be a contiguous fp16 / bf16 GPU tensor")
    b_ptr, b_period, b_value = None, 1, 0.0
    if isinstance(b, torch.Tensor):
        _check(b, "b", a.dtype)
        if not b.is_contiguous():
            raise ValueError("b must be contiguous")
        shape = list(b.shape)
        while shape and shape[0] == 1:
            shape.pop(0)
        if shape != list(a.shape)[len(a.shape) - len(shape):]:
            raise ValueError(f"b of shape {tuple(b.shape)} does not broadcast over the leading dims of {tuple(a.shape)}")
        b_ptr, b_period = _p(b), max(1, b.numel())
    elif b is not None:
        b_value = float(b)
    if out is None:
        out = torch.empty_like(a)
    else:
        _check(out, "out", a.dtype)
        _check_out(out, a.numel(), "a.numel()")
    rc = lib.aitamd_elementwise(fid, _TORCH_DTYPE_ID[a.dtype], _p(a), b_ptr, _p(out), a.numel(), b_period, b_value, swap,
                                _stream_ptr())
    _kernels.check(rc, f"elementwise({func})")
    return out


def split(x: torch.Tensor, sizes, dim: int) -> Tuple[torch.Tensor, ...]:
    """torch.split(x, sizes, dim) with every piece a new contiguous tensor, one strided row copy per piece
    (python/aitemplate/compiler/ops/tensor/split.py:31-170)."""
    lib = _kernels.load()
    if not x.is_cuda or not x.is_contiguous():
        raise ValueError("x must be a contiguous GPU tensor")
    dim %= x.dim()
    if sum(sizes) != x.shape[dim]:
        raise ValueError(f"split sizes {list(sizes)} do not add up to {x.shape[dim]}")
    rows = 1
    for d in x.shape[:dim]:
        rows *= d
    inner = x.element_size()
    for d in x.shape[dim + 1:]:
        inner *= d
    outs, start = [], 0
    for n in sizes:
        o = torch.empty(*x.shape[:dim], n, *x.shape[dim + 1:], dtype=x.dtype, device=x.device)
        rc = lib.aitamd_copy_rows(ctypes.c_void_p(x.data_ptr() + start * inner), _p(o), rows, n * inner, x.shape[dim] * inner, n * inner,
                                  _stream_ptr())
        _kernels.check(rc, "split")
        outs.append(o)
        start += n
    return tuple(outs)


def concatenate(tensors, dim: int) -> torch.Tensor:
    """torch.cat(tensors, dim) as one strided row copy per input
    (python/aitemplate/compiler/ops/tensor/concatenate.py:31-170)."""
    lib = _kernels.load()
    first = tensors[0]
    dim %= first.dim()
    for t in tensors:
        if not t.is_cuda or not t.is_contiguous() or t.dtype != first.dtype:
            raise ValueError("inputs must be contiguous GPU tensors of one dtype")
        if list(t.shape[:dim]) + list(t.shape[dim + 1:]) != list(first.shape[:dim]) + list(first.shape[dim + 1:]):
            raise ValueError("inputs differ in a dim other than the concatenated one")
    total = sum(t.shape[dim] for t in tensors)
    out = torch.empty(*first.shape[:dim], total, *first.shape[dim + 1:], dtype=first.dtype, device=first.device)
    rows = 1
    for d in first.shape[:dim]:
        rows *= d
    inner = first.element_size()
    for d in first.shape[dim + 1:]:
        inner *= d
    start = 0
    for t in tensors:
        n = t.shape[dim]
        rc = lib.aitamd_copy_rows(_p(t), ctypes.c_void_p(out.data_ptr() + start * inner), rows, n * inner, n * inner, total * inner,
                                  _stream_ptr())
        _kernels.check(rc, "concatenate")
        start += n
    return out


# ---- the attention block of a decoder that is being served ------------------------------------------------------
# Launches go to the stream that is current on the operands' device; every tensor has to be on that device.

def _operands(*named) -> torch.device:
    """The device of the tensors in (name, tensor or None, dtypes or None) triples, checked: one GPU, the types given."""
    device = None
    for name, t, dtypes in named:
        if t is None:
            continue
        _check(t, name)
        if dtypes is not None and t.dtype not in dtypes:
            raise ValueError(f"{name}: dtype {t.dtype} is not {' or '.join(str(d) for d in dtypes)}")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
    return device


def _dense_heads(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t


def quantize_rows(x: torch.Tensor, out: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of `x` [..., columns] (fp16 / bf16) as 8-bit integers, and one fp32 scale a row ([...]): scale = max|x| / 127 and
    the whole number nearest to x / scale (of 127 x / max|x|, exactly; ties to even).  A row of zeros has scale 0; a row
    with an infinity or a NaN has scale NaN and zeros.  `x` may be a 2-D view with row pitch."""
    if out is None and scale is None:
        result = _native_decoder.quantize_rows(x)
        if result is not NotImplemented:
            return result
    device = _operands(("x", x, tuple(_TORCH_DTYPE_ID)), ("out", out, (torch.int8,)), ("scale", scale, (torch.float32,)))
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    lead, columns = x.shape[:-1], x.shape[-1]
    rows = 1
    for d in lead:
        rows *= d
    ldx = _row_pitch(x, "x") if x.dim() == 2 else columns
    if x.dim() != 2 and not x.is_contiguous():
        raise ValueError("x must be contiguous, or 2-D with a contiguous last dimension")
    if rows > 1 and ldx < columns:
        raise ValueError("x: rows overlap")
    if out is None:
        out = torch.empty(x.shape, dtype=torch.int8, device=device)
    else:
        _check_out(out, rows * columns, "x.numel()")
    if scale is None:
        scale = torch.empty(lead, dtype=torch.float32, device=device)
    else:
        _check_out(scale, rows, "rows")
    with torch.cuda.device(device):
        rc = _kernels.load().aitamd_quantize_rows(_TORCH_DTYPE_ID[x.dtype], _p(x), _p(out), _p(scale), rows, columns, ldx, columns,
                                                  _stream_ptr())
    _kernels.check(rc, "quantize_rows")
    return out, scale


def gemm_int8_workspace_bytes(M: int, N: int, K: int, bias: bool = False, dtype=torch.float16, algo: int = -1,
                              any_byte: bool = False) -> int:
    """Bytes of scratch memory with which `gemm_rcr_int8` may choose any of its instances for this problem (0: none takes any).
    `any_byte`: operands that are views at any pitch and address, whose rows may be no whole dwords (they are laid out there first)."""
    lib = _kernels.load()
    need = int(lib.aitamd_gemm_int8_workspace_bytes(_TORCH_DTYPE_ID[dtype], algo, int(bool(bias)), M, N, K))
    return max(need, int(lib.aitamd_gemm_int8_layout_bytes(M, N, K))) if any_byte else need


def _off_dwords(t: torch.Tensor, name: str) -> bool:
    """Whether the rows of an 8-bit operand are no whole dwords."""
    rows, columns = t.shape
    return (columns | t.data_ptr() | (_row_pitch(t, name) if rows > 1 else 0)) % 4 != 0


def gemm_rcr_int8(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  dtype=torch.float16, out: Optional[torch.Tensor] = None, algo: int = -1,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = a_scale * b_scale * (a @ b.T) (+ bias) of 8-bit integers `a` [..., K] with a fp32 scale for each row ([...], see
    `quantize_rows`) and `b` [N, K] with one for each of its rows ([N]: a layer's output channels); `out` and `bias` [N] are of
    type `dtype`.  The sums are exact, K goes up to 131071, rows may lie at any byte.  `a` and `b` may have row pitch (2-D views);
    `algo` and `workspace` as of `gemm` (sizes from `gemm_int8_workspace_bytes`); without one, rows that are no whole dwords have
    theirs for the call."""
    if dtype not in _TORCH_DTYPE_ID:
        raise ValueError(f"unsupported dtype {dtype}")
    result = _native_decoder.gemm_rcr_int8(a, b, a_scale, b_scale, bias, dtype is torch.bfloat16, out, algo, workspace)
    if result is not NotImplemented:
        return result
    device = _operands(("a", a, (torch.int8,)), ("b", b, (torch.int8,)), ("a_scale", a_scale, (torch.float32,)),
                       ("b_scale", b_scale, (torch.float32,)), ("bias", bias, (dtype,)), ("out", out, (dtype,)),
                       ("workspace", workspace, (torch.uint8,)))
    if a.dim() < 1:
        raise ValueError("a must have at least one dimension")
    lead, K = a.shape[:-1], a.shape[-1]
    M = 1
    for d in lead:
        M *= d
    if b.dim() != 2 or b.shape[1] != K:
        raise ValueError(f"b must be [N, K={K}], got {tuple(b.shape)}")
    N = b.shape[0]
    a2 = a if a.dim() == 2 else a.reshape(M, K)
    for t, n, name in ((a_scale, M, "a_scale"), (b_scale, N, "b_scale")) + (((bias, N, "bias"),) if bias is not None else ()):
        if t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous with {n} elements, got shape {tuple(t.shape)}")
    if out is None:
        out = torch.empty(*lead, N, dtype=dtype, device=device)
    if out.dim() == 2 and out.shape == (M, N) and (out.stride(1) == 1 or N == 1) and out.stride(0) >= N:
        out2 = out  # (rows of a wider buffer: written in place)
    else:
        _check_out(out, M * N, "M*N")
        out2 = out.view(M, N)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 GPU tensor (see new_workspace)")
    with torch.cuda.device(device):
        odd_a, odd_b = _off_dwords(a2, "a"), _off_dwords(b, "b")
        if workspace is None and algo < 0 and (odd_a or odd_b):
            # (an operand whose rows are no whole dwords is laid out there first; nothing in it has to be zero for that)
            need = int(_kernels.load().aitamd_gemm_int8_layout_bytes(M if odd_a else 0, N if odd_b else 0, K))
            workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        rc = _kernels.load().aitamd_gemm_rcr_int8(
            _TORCH_DTYPE_ID[dtype], algo, _p(a2), _p(b), _p(a_scale), _p(b_scale), _p(bias), _p(out2), M, N, K, _row_pitch(a2, "a"),
            _row_pitch(b, "b"), _row_pitch(out2, "out"), _p(workspace), 0 if workspace is None else workspace.numel(), _stream_ptr())
    _kernels.check(rc, "gemm_rcr_int8")
    return out


def rotary_frequencies(rotated: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, low: float = 1.0, high: float = 32.0,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """(freqs, scale) for `rotary_embedding`: base ** (-2 i / rotated) for pair i, in fp32 on `device`, and the factor of the result.

    `scaling` stretches them for contexts `factor` times as long as the `original_length` that a model was trained on:

    * None: as they are;
    * "linear": every frequency divided by `factor`;
    * "base": the base raised to base * factor ** (rotated / (rotated - 2)), which divides the lowest frequency by `factor`
      and leaves the highest;
    * "bands": frequencies that turn fewer than `low` times over `original_length` are divided by `factor`, those that turn
      more than `high` times stay, and in between the share that stays grows evenly with the number of turns;
    * "yarn": likewise, but the share grows evenly with the pair's index, between the pairs of `high` and of `low` turns
      (rounded outwards), and the result is scaled by 0.1 ln(factor) + 1."""
    import math

    if rotated < 2 or rotated % 2:
        raise ValueError(f"rotated must be an even number of at least 2, got {rotated}")
    if scaling not in (None, "linear", "base", "bands", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not base > 1.0 or (scaling is not None and not factor >= 1.0):
        raise ValueError(f"base {base} must be above 1 and factor {factor} at least 1")
    if scaling in ("bands", "yarn") and (not original_length or original_length <= 0 or not 0.0 < low < high):
        raise ValueError(f"{scaling!r} needs original_length and 0 < low < high")
    if scaling == "base" and rotated == 2:
        raise ValueError("'base' needs more than one pair")
    pair = torch.arange(rotated // 2, dtype=torch.float64, device="cpu")
    if scaling == "base":
        base = base * factor ** (rotated / (rotated - 2))
    freqs = base ** (pair * (-2.0 / rotated))
    scale = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling in ("bands", "yarn"):
        if scaling == "bands":
            turns = original_length * freqs / (2.0 * math.pi)
            stays = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        else:
            def pair_of(turns):  # the (fractional) pair that turns so often
                return rotated / 2.0 * math.log(original_length / (turns * 2.0 * math.pi)) / math.log(base)

            first = max(math.floor(pair_of(high)), 0)
            last = min(math.ceil(pair_of(low)), rotated - 1)
            stays = 1.0 - ((pair - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
            scale = 0.1 * math.log(factor) + 1.0
        freqs = freqs * stays + freqs / factor * (1.0 - stays)
    return freqs.float().to(device), scale


def _check_freqs(freqs: torch.Tensor, head_dim: int) -> int:
    if freqs.dim() != 1 or not freqs.is_contiguous() or 2 * freqs.numel() > head_dim:
        raise ValueError(f"freqs must be a contiguous 1-D tensor of at most head_dim / 2 = {head_dim // 2} numbers, got shape {tuple(freqs.shape)}")
    return 2 * freqs.numel()


def rotary_embedding(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
                     inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions: `x` [tokens, heads, head_dim] or [batch, seq, heads, head_dim] (any strides, contiguous head dims) with the
    first 2 len(freqs) dims of every head turned by positions * freqs: dims i and len(freqs) + i, or with `interleaved` 2 i and
    2 i + 1, become scale * (x1 cos - x2 sin, x2 cos + x1 sin); the other dims are handed through.

    `positions`: int32 or int64 [tokens], [batch, seq], or [seq] for every batch entry.  `freqs`: fp32, see `rotary_frequencies`
    (whose second result is `scale`).  `inverse` turns back: the gradient with respect to `x` of the same call without it.
    `out` may be `x` itself and must not overlap it otherwise."""
    result = _native_decoder.rotary_embedding(x, positions, freqs, interleaved, scale, inverse, out)
    if result is not NotImplemented:
        return result
    device = _operands(("x", x, tuple(_TORCH_DTYPE_ID)), ("positions", positions, (torch.int32, torch.int64)),
                       ("freqs", freqs, (torch.float32,)), ("out", out, (x.dtype,)))
    if x.dim() not in (3, 4):
        raise ValueError("x must be [tokens, heads, head_dim] or [batch, seq, heads, head_dim]")
    rotated = _check_freqs(freqs, x.shape[-1])
    if tuple(positions.shape) not in (tuple(x.shape[:-2]), tuple(x.shape[-3:-2])):
        raise ValueError(f"positions of shape {tuple(positions.shape)} do not fit x of shape {tuple(x.shape)}")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=device)
    elif out.shape != x.shape:
        raise ValueError(f"out must be {tuple(x.shape)}, got {tuple(out.shape)}")
    _dense_heads(x, "x"), _dense_heads(out, "out")
    flat = x.dim() == 3
    batch, seq = (1, x.shape[0]) if flat else (x.shape[0], x.shape[1])
    xs, os = ((0,) + t.stride() if flat else t.stride() for t in (x, out))
    ps = (0, positions.stride(0)) if positions.dim() == 1 else positions.stride()
    with torch.cuda.device(device):
        rc = _kernels.load().aitamd_rotary_embedding(
            _TORCH_DTYPE_ID[x.dtype], _p(x), _p(out), _p(positions), int(positions.dtype == torch.int64), _p(freqs), batch, seq,
            x.shape[-2], x.shape[-1], rotated, *xs[:3], *os[:3], *ps, float(scale), int(bool(interleaved)), int(bool(inverse)),
            _stream_ptr())
    _kernels.check(rc, "rotary_embedding")
    return out


def _paged_cache(k_cache, v_cache, block_table, lengths, offsets, tokens, head_dim) -> "_kernels.PagedCache":
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache must be [pages, page_size, kv_heads, head_dim], got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)}")
    pages, page_size, kv_heads, dim = k_cache.shape
    if dim != head_dim:
        raise ValueError(f"head_dim of the cache is {dim}, of the operands {head_dim}")
    _dense_heads(k_cache, "k_cache"), _dense_heads(v_cache, "v_cache")
    if lengths.dim() != 1 or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous 1-D tensor")
    batch = lengths.numel()
    if block_table.dim() != 2 or block_table.shape[0] != batch or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be [batch = {batch}, pages of a sequence] with contiguous rows, got {tuple(block_table.shape)}")
    if offsets is not None and (offsets.dim() != 1 or not offsets.is_contiguous() or offsets.numel() != batch + 1):
        raise ValueError(f"offsets must be a contiguous 1-D tensor of batch + 1 = {batch + 1} entries")
    if offsets is None and tokens != batch:
        raise ValueError(f"without offsets every sequence has one row: {tokens} rows, {batch} sequences")
    return _kernels.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), pages, page_size, kv_heads, dim, *k_cache.stride()[:3],
                               *v_cache.stride()[:3], block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                               lengths.data_ptr(), None if offsets is None else offsets.data_ptr(), batch, tokens)


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, offsets: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                    freqs: Optional[torch.Tensor] = None, interleaved: bool = False, scale: float = 1.0, first_position: int = 0,
                    q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """One step's keys and values `k`, `v` [tokens, kv_heads, head_dim] into the pages of their sequences, in one launch with the
    rotation of the keys and of the queries `q` [tokens, heads, head_dim]; returns the rotated queries (None without `q`).

    `k_cache`, `v_cache` [pages, page_size, kv_heads, head_dim], any strides with contiguous head dims: a cache that lies head by
    head is passed transposed.  `block_table` [batch, n] int32: the pages of each sequence in order; entries outside [0, pages)
    are no page.  `lengths` [batch] int32: tokens that the sequences have in their pages before the step.  `offsets` [batch + 1]
    int32: sequence i has the rows offsets[i] to offsets[i + 1]; without it, row i.  Row j of a sequence goes to its place
    lengths[i] + j, rotated (with `freqs`, as by `rotary_embedding`) for position first_position + lengths[i] + j.

    Rows from offsets[batch] on are left as they were, in `q_out` too; keys and values that no page is there for are dropped.
    Pages that are written must not be shared between sequences.  `lengths` stay as they are: the attention of the same step
    takes them as they are too.  `q_out` may be `q`."""
    result = _native_decoder.paged_kv_append(k, v, k_cache, v_cache, block_table, lengths, offsets, q, freqs, interleaved, scale,
                                             first_position, q_out)
    if result is not NotImplemented:
        return result
    types = tuple(_TORCH_DTYPE_ID)
    device = _operands(("k", k, types), ("v", v, (k.dtype,)), ("k_cache", k_cache, (k.dtype,)), ("v_cache", v_cache, (k.dtype,)),
                       ("block_table", block_table, (torch.int32,)), ("lengths", lengths, (torch.int32,)),
                       ("offsets", offsets, (torch.int32,)), ("q", q, (k.dtype,)), ("freqs", freqs, (torch.float32,)),
                       ("q_out", q_out, (k.dtype,)))
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"k and v must be [tokens, kv_heads, head_dim], got {tuple(k.shape)} and {tuple(v.shape)}")
    tokens, kv_heads, head_dim = k.shape
    cache = _paged_cache(k_cache, v_cache, block_table, lengths, offsets, tokens, head_dim)
    if cache.kv_heads != kv_heads:
        raise ValueError(f"the cache has {cache.kv_heads} heads, k {kv_heads}")
    _dense_heads(k, "k"), _dense_heads(v, "v")
    rotated = 0 if freqs is None else _check_freqs(freqs, head_dim)
    q_in, heads, qs, os = None, 0, (0, 0), (0, 0)
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
    else:
        if q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != head_dim:
            raise ValueError(f"q must be [{tokens}, heads, {head_dim}], got {tuple(q.shape)}")
        _dense_heads(q, "q")
        if q_out is None and rotated == 0:
            q_out = q  # (nothing is done to it)
        elif q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
        elif q_out.shape != q.shape:
            raise ValueError(f"q_out must be {tuple(q.shape)}, got {tuple(q_out.shape)}")
        _dense_heads(q_out, "q_out")
        if q_out is not q or rotated:
            q_in, heads, qs, os = q, q.shape[1], q.stride(), q_out.stride()
    with torch.cuda.device(device):
        rc = _kernels.load().aitamd_paged_kv_append(
            _TORCH_DTYPE_ID[k.dtype], cache, _p(k), *k.stride()[:2], _p(v), *v.stride()[:2], _p(q_in), *qs[:2],
            _p(q_out) if q_in is not None else None, *os[:2], heads, _p(freqs) if rotated else None, rotated, int(first_position),
            float(scale), int(bool(interleaved)), _stream_ptr())
    _kernels.check(rc, "paged_kv_append")
    return q_out


def prefix_attention_workspace_bytes(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                                     lengths: torch.Tensor, offsets: Optional[torch.Tensor] = None, prefix_length: int = 0) -> int:
    """Bytes of scratch memory that `prefix_attention` of these arguments needs."""
    cache = _paged_cache(k_cache, v_cache, block_table, lengths, offsets, q.shape[0], q.shape[-1])
    with torch.cuda.device(q.device):
        need = int(_kernels.load().aitamd_prefix_attention_workspace_bytes(cache, q.shape[1], int(prefix_length)))
    if need < 0:
        raise RuntimeError(f"prefix_attention failed: {_kernels.last_error()}")
    return need


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                     offsets: Optional[torch.Tensor] = None, prefix_table: Optional[torch.Tensor] = None, prefix_length: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one step's queries `q` [tokens, heads, head_dim] over a paged cache, after `paged_kv_append` of the same step
    (`k_cache`, `v_cache`, `block_table`, `lengths`, `offsets` as there, `lengths` still those from before the step).

    Every row sees the first `prefix_length` keys of the pages `prefix_table` [n] int32, which the whole batch shares, and those of
    its own sequence's pages up to itself.  Query head h reads key head h // (heads / kv_heads).  `scale` is head_dim ** -0.5
    unless given.  In fp16, keys of less than 2^-33 of the weight of a row's largest count as none.  Rows that see no key are zeros;
    rows of `out` from offsets[batch] on are left as they were.  What lies in a page behind a sequence's last key may be anything;
    keys and values of the step's later rows do not count for a row, as long as they are finite.

    Without `offsets`, or with up to 32 rows a sequence on average (a token has heads / kv_heads of them for each key head), the prefix
    is read once for every 128 rows of the whole batch; otherwise, and for one sequence alone, once for every tile of a sequence's
    own rows, where a sequence of one token beside prompts has a tile for itself.

    page_size has to be a multiple of 16, head_dim one of 8 up to 256.  `workspace`: a buffer from `new_workspace` of
    `prefix_attention_workspace_bytes`, allocated for the call otherwise; calls that may overlap in time need one each."""
    result = _native_decoder.prefix_attention(q, k_cache, v_cache, block_table, lengths, offsets, prefix_table, prefix_length, scale, out,
                                              workspace)
    if result is not NotImplemented:
        return result
    device = _operands(("q", q, tuple(_TORCH_DTYPE_ID)), ("k_cache", k_cache, (q.dtype,)), ("v_cache", v_cache, (q.dtype,)),
                       ("block_table", block_table, (torch.int32,)), ("lengths", lengths, (torch.int32,)),
                       ("offsets", offsets, (torch.int32,)), ("prefix_table", prefix_table, (torch.int32,)), ("out", out, (q.dtype,)),
                       ("workspace", workspace, (torch.uint8,)))
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    tokens, heads, head_dim = q.shape
    cache = _paged_cache(k_cache, v_cache, block_table, lengths, offsets, tokens, head_dim)
    if prefix_table is not None and (prefix_table.dim() != 1 or not prefix_table.is_contiguous()):
        raise ValueError("prefix_table must be a contiguous 1-D tensor")
    if prefix_length and prefix_table is None:
        raise ValueError("prefix_length without prefix_table")
    _dense_heads(q, "q")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    elif out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    _dense_heads(out, "out")
    lib = _kernels.load()
    with torch.cuda.device(device):
        if workspace is None:
            need = int(lib.aitamd_prefix_attention_workspace_bytes(cache, heads, int(prefix_length)))
            workspace = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        elif not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 GPU tensor (see new_workspace)")
        rc = lib.aitamd_prefix_attention(
            _TORCH_DTYPE_ID[q.dtype], cache, _p(q), *q.stride()[:2], _p(out), *out.stride()[:2], heads, _p(prefix_table),
            0 if prefix_table is None else prefix_table.numel(), int(prefix_length),
            float(head_dim ** -0.5 if scale is None else scale), _p(workspace), 0 if workspace is None else workspace.numel(), _stream_ptr())
    _kernels.check(rc, "prefix_attention")
    return out
