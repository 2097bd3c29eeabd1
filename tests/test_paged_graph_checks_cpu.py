"""What the graph ops paged_kv_append and prefix_attention check of the tensors that their kernels follow, without a GPU: at the
construction of the graph what its shapes tell, at a run (the generated functions, compiled for the host with entry points that launch
nothing) what only a run knows."""
import ctypes
import os
import subprocess

import pytest

from aitemplate_amd.backend import registry
from aitemplate_amd.compiler import ops
from aitemplate_amd.frontend import IntVar
from test_decoder_ops_cpu import cache, generated, tensor

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STUBS = """
#include <stdio.h>
#include "aitemplate_amd_kernels.h"
static int launches = 0;
extern "C" int stub_launches() { return launches; }
extern "C" const char* aitamd_last_error() { return ""; }
extern "C" int aitamd_gemm_find_algo(int, int, const char*) { return -1; }
extern "C" int aitamd_paged_kv_append(int, const aitamd_paged_cache*, const void*, int64_t, int64_t, const void*, int64_t, int64_t,
                                      const void*, int64_t, int64_t, void*, int64_t, int64_t, int64_t, const float*, int64_t, int64_t,
                                      float, int, void*) { return ++launches, 0; }
extern "C" int aitamd_prefix_attention(int, const aitamd_paged_cache*, const void*, int64_t, int64_t, void*, int64_t, int64_t, int64_t,
                                       const int32_t*, int64_t, int64_t, float, void*, int64_t, void*) { return ++launches, 0; }
"""


def operands(batch, ends, tokens=None):
    t = tokens or IntVar(values=[1, 64], name="t")
    q, k, v = tensor("q", [t, 8, 64]), tensor("k", [t, 2, 64]), tensor("v", [t, 2, 64])
    table, lengths = tensor("table", [batch, 9], "int32"), tensor("lengths", [batch], "int32")
    return q, k, v, table, lengths, tensor("offsets", [ends], "int32"), tensor("f", [32], "float32")


def append(batch, ends):
    q, k, v, table, lengths, offsets, freqs = operands(batch, ends)
    op = ops.paged_kv_append()
    op(q, k, v, *cache(), table, lengths, freqs, offsets)
    return op


def attention(batch, ends):
    q, _, _, table, lengths, offsets, _ = operands(batch, ends)
    op = ops.prefix_attention()
    op(q, *cache(), table, lengths, offsets)
    return op


def dim(low, high, name):
    return low if low == high else IntVar(values=[low, high], name=name)


@pytest.mark.parametrize("make", [append, attention])
@pytest.mark.parametrize("batch,ends,fits", [((8, 8), (9, 9), True), ((8, 8), (8, 8), False), ((8, 8), (2, 2), False), ((8, 8), (2, 9), True),
                                             ((8, 8), (2, 8), False), ((1, 8), (2, 9), True), ((1, 8), (2, 2), True), ((2, 8), (2, 2), False),
                                             ((1, 8), (10, 20), False), ((1, 8), (9, 20), True)])
def test_offsets_that_no_batch_has(make, batch, ends, fits):
    batch, ends = dim(*batch, "b"), dim(*ends, "e")
    if fits:
        make(batch, ends)
    else:
        with pytest.raises(RuntimeError, match="offsets"):
            make(batch, ends)


@pytest.mark.parametrize("make", [append, attention])
def test_offsets_of_another_batch_at_a_run(make, tmp_path):
    # up to 8 sequences, offsets that are always two (or any number): the run has to fit
    op = make(IntVar(values=[1, 8], name="b"), IntVar(values=[2, 9], name="e"))
    source, _, call = generated(op, "op")
    names = call.strip()[len("op("):-2].split(", ")
    # the model's members, as the call names them, and a call that says what it threw
    pointers = [n for n in names if n in {t._attrs["name"] for t in op._attrs["inputs"] + op._attrs["outputs"]}]
    dims = [n for n in names if n in ("t", "b", "e", "pages")]
    assert "b" in dims and "e" in dims
    main = "\n".join([STUBS, source, 'extern "C" int run(int64_t t, int64_t b, int64_t e, char* what, int64_t n) {', "  char memory[64] = {};",
                      *[f"  void* {n} = memory;" for n in pointers], "  int64_t pages = 4;",
                      *[f"  int64_t {n} = 9;" for n in set(names) - set(pointers) - set(dims) - {"stream", "nullptr", "0", "workspace_", "workspace_size_"}],
                      "  uint8_t* workspace_ = nullptr; int64_t workspace_size_ = 4096; hipStream_t stream = nullptr;",
                      "  (void)workspace_, (void)workspace_size_, (void)pages, (void)t;",
                      f"  try {{ ait::{call.strip()} }} catch (const std::exception& x) {{ snprintf(what, n, \"%s\", x.what()); return 1; }}",
                      "  return 0;", "}"])
    (tmp_path / "op.cpp").write_text(main)
    # (-Bsymbolic: its own entry points, also where the library of the same names is loaded)
    subprocess.run(["g++", "-O0", "-std=c++17", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT}/include", "-I/opt/rocm/include",
                    str(tmp_path / "op.cpp"), "-o", str(tmp_path / "op.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "op.so"))
    lib.run.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_char_p, ctypes.c_int64]
    what = ctypes.create_string_buffer(256)
    for batch, ends in [(8, 2), (8, 8), (1, 9), (3, 5)]:
        before = lib.stub_launches()
        assert lib.run(20, batch, ends, what, 256) == 1 and b"offsets" in what.value, (batch, ends)
        assert lib.stub_launches() == before
    for batch, ends in [(8, 9), (1, 2)]:
        before = lib.stub_launches()
        assert lib.run(20, batch, ends, what, 256) == 0 and lib.stub_launches() == before + 1
