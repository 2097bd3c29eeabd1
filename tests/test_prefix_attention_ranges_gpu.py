"""Attention over a paged cache on the GPU where many keys have weights far below a row's largest: one by one next to nothing, together
not.  In all shapes: one sequence in parts, a batch that decodes, its prefix in tiles of 128 rows, prompts.

Tolerance, with eps the type's step, y the result: the weights are rounded by eps / 2, their sum is taken of the rounded ones, the result
is rounded once: 3 eps / 2 |y| (v > 0 here).  A score is off by 64 2^-24 of its size at most, an exponential by 2^-22, both twice, in a
weight and in the sum; a sum of n equal numbers in 32 bits, taken in runs of 16 and more, by n / 16 2^-24.  In fp16 weights are held 2^8
times as large as they are, against a reference point that is at most the row's largest: off by 2^-25 / 2^8 = 2^-33 of the largest
each where they are small, n 2^-33 |v| for n of them."""
import math

import pytest
import torch

from aitemplate_amd import eager
from paged_common import DEV

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def tail(dtype, orders, keys, batch, tokens, heads, first):
    """`tokens` rows a sequence over a prefix of `keys` keys that are 2^-orders of one key's weight, which is the first of all or in the
    middle of them; one key of that kind for each row of its own.  All pages of such keys are one."""
    D, page = 64, 16
    k, v = (torch.zeros(2, page, heads, D, dtype=dtype, device=DEV) for _ in range(2))
    v[:] = torch.linspace(0.5, 1.5, D, device=DEV).to(dtype)
    # scale ln 2: scores of 0 and of `orders` are weights of 1 and of 2^orders
    k[0, 3, :, 0] = orders
    v[0, 3] = 0.0
    q = torch.zeros(batch * tokens, heads, D, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    table = torch.ones(1, -(-tokens // page), dtype=torch.int32, device=DEV).expand(batch, -1)
    prefix_table = torch.ones(keys // page, dtype=torch.int32, device=DEV)
    prefix_table[0 if first else len(prefix_table) // 2] = 0
    offsets = torch.arange(0, batch * tokens + 1, tokens, dtype=torch.int32, device=DEV) if tokens > 1 else None
    got = eager.prefix_attention(q, k, v, table, torch.zeros(batch, dtype=torch.int32, device=DEV), offsets, prefix_table=prefix_table,
                                 prefix_length=keys, scale=math.log(2.0))
    seen = (keys - 1 + torch.arange(1, tokens + 1, device=DEV).double()).repeat(batch)
    weight = seen * 2.0 ** -orders
    want = (weight / (1.0 + weight))[:, None] * v[1, 0, 0].double()
    eps = torch.finfo(dtype).eps / 2
    allowed = want * (3 * eps + 64 * orders * 2.0 ** -23 + 2.0 ** -21 + keys / 16 * 2.0 ** -24) * 1.01
    if dtype == torch.float16:
        allowed = allowed + seen[:, None] * 2.0 ** -33 * v[1, 0, 0].double()
    off = (got.double() - want[:, None]).abs() / allowed[:, None]
    assert off.max() <= 1.0, (off.max().item(), got[0, 0, :3], want[0, :3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("orders", [25.5, 27.0, 30.0])
@pytest.mark.parametrize("batch,tokens,heads", [(1, 1, 1), (512, 1, 1), (3, 1, 8), (1, 1024, 64), (2, 129, 4)])
def test_many_keys_far_below_the_largest(dtype, first, orders, batch, tokens, heads):
    tail(dtype, orders, 1 << 17, batch, tokens, heads, first)
