"""Attention over a paged cache on the GPU in the shapes that take tiles of 128 rows (prompts, the prefix of a batch that decodes),
with scores that have a tile's fast form taken back: scales, maxima that jump between the tiles of 64 keys, NaN and infinite scores in
and behind the first tile.  Tolerance: see test_prefix_attention_gpu.py."""
import math

import pytest
import torch

from paged_common import DEV, Paged
from test_prefix_attention_gpu import attend, check, one_sequence, operands

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def prompt(dtype):
    return Paged(dtype, [700, 20], [300, 257], 2, 64, 16, 0, ragged=True), 4


def prompt_behind_a_prefix(dtype):
    return Paged(dtype, [100, 33], [150, 257], 1, 80, 32, 500, ragged=True), 3


def decoding(dtype):
    return Paged(dtype, [700, 20, 130, 0] * 5, [1] * 20, 2, 96, 16, 777), 8


SHAPES = [prompt, prompt_behind_a_prefix, decoding]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 20.0])
def test_scales(dtype, shape, scale):
    c, heads = shape(dtype)
    q = operands(c, heads, c.k.shape[2], c.k.shape[3])
    check(c, q, attend(c, q, scale=scale), scale)


def places(c):
    """(page, place in it, place among the prefix's or the sequence's own keys) of every key."""
    for pages, count in [(c.prefix_table, c.prefix)] + [(c.table[i], p + n) for i, (p, n) in enumerate(zip(c.past, c.new))]:
        place = torch.arange(count, device=DEV)
        yield pages[place // c.page].long(), place % c.page, place


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("largest", [-1, 1, 2, 3])
def test_maxima_that_jump_from_tile_to_tile(dtype, shape, largest):
    # keys 4 times as large from one run of 64 to the next up to a run (largest), or to the last, and small ones behind it: the
    # largest score of a run is tens of binary orders above the runs' before it
    c, heads = shape(dtype)
    q = operands(c, heads, c.k.shape[2], c.k.shape[3])
    for page, at, place in places(c):
        run = place // 64
        size = 0.25 * 4.0 ** run.clamp(max=3).double()
        if largest >= 0:
            size = torch.where(run <= largest, size, 0.25)
        c.k[page, at] = (c.k[page, at].double() * size[:, None, None]).to(dtype)
    check(c, q, attend(c, q, scale=1.0), 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("place", [0, 70, 130, 200, 319])
def test_nan_and_infinite_scores_behind_the_first_tile(dtype, shape, place):
    c, heads = shape(dtype)
    kv_heads, group = c.k.shape[2], heads // c.k.shape[2]
    q = operands(c, heads, kv_heads, c.k.shape[3])
    # of the prefix where there is one, otherwise of the first sequence, whose rows all see it
    pages = c.prefix_table if c.prefix else c.table[0]
    rows = slice(0, c.tokens) if c.prefix else slice(0, c.new[0])
    at = pages[place // c.page].long(), place % c.page
    clean = attend(c, q)
    touched = torch.zeros(c.tokens, heads, dtype=torch.bool, device=DEV)
    touched[rows, :group] = True

    held = c.k[at].clone()
    c.k[at][0, 5] = math.nan
    got = attend(c, q)
    assert torch.isnan(got[touched]).all() and torch.equal(got[~touched], clean[~touched])

    # an infinity takes the whole weight (infinity - infinity) or none at all, as q's sign says
    c.k[at].copy_(held)
    q[:, :, 5] = torch.where(q[:, :, 5] >= 0, 1.0, -1.0).to(dtype)
    c.k[at][0, 5] = math.inf
    got = attend(c, q)
    up = touched & (q[:, :, 5] > 0)
    assert torch.isnan(got[up]).all() and torch.isfinite(got[~up]).all()
    # ... none: as the formula has it without that key.  (Rows with NaN have their wave's other rows take the full form, with another
    # reference point than the fast form's: the same within the tolerance, not bit for bit.)
    shared = [c.read(t, c.prefix_table, c.prefix) for t in (c.k, c.v)]
    for i, (p, n) in enumerate(zip(c.past, c.new)):
        if c.prefix or i == 0:
            mine = slice(c.starts[i], c.starts[i + 1])
            k, v = (torch.cat((s, c.read(t, c.table[i], p + n))) for s, t in zip(shared, (c.k, c.v)))
            k[place] = 0.0
            hidden = torch.arange(k.shape[0], device=DEV) >= c.prefix + torch.arange(p + 1, p + n + 1, device=DEV)[:, None]
            hidden[:, place] = True
            want, allowed = one_sequence(q[mine], k, v, hidden, q.shape[2] ** -0.5, dtype)
            down = (q[mine, :, 5] < 0) & touched[mine]
            assert ((got[mine].double() - want).abs() <= allowed)[down].all()
