"""paged_kv_append writes its cache in place: no constant of the model, which all of its runtimes share, without a GPU."""
import pytest
import torch

from aitemplate_amd.compiler import ops
from aitemplate_amd.frontend import IntVar, Tensor
from test_decoder_ops_cpu import cache, tensor


@pytest.mark.parametrize("which", [(0,), (1,), (0, 1)])
@pytest.mark.parametrize("bound", [False, True])
def test_a_constant_cache_is_refused(which, bound):
    b = IntVar(values=[1, 8], name="b")
    q, k, v = tensor("q", [b, 8, 64]), tensor("k", [b, 2, 64]), tensor("v", [b, 2, 64])
    table, lengths, freqs = tensor("table", [b, 3], "int32"), tensor("lengths", [b], "int32"), tensor("f", [32], "float32")
    ops.paged_kv_append()(q, k, v, *cache(), table, lengths, freqs)
    caches = [tensor(n, [4, 16, 2, 64]) for n in ("k_cache", "v_cache")]
    for i in which:
        caches[i] = Tensor([4, 16, 2, 64], dtype="float16", name=f"constant_{i}")
        if bound:
            from aitemplate_amd.compiler.base import ConstantTensorData

            caches[i]._bind_data(ConstantTensorData.from_torch(torch.zeros(4, 16, 2, 64, dtype=torch.float16)))
    with pytest.raises(RuntimeError, match="must be an input of the model"):
        ops.paged_kv_append()(q, k, v, *caches, table, lengths, freqs)
    # what only reads a cache may have a constant one
    ops.prefix_attention()(q, *caches, table, lengths)
