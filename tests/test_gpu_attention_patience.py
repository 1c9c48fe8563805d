"""Rows that attend to NaN are gone over a second time, position by position, which takes seconds on a long cache.  Whoever waits meanwhile
-- the same CTA's other warps, already at the next unit, and in a pair the other CTA -- waits as long as that pass moves on.

Tolerance of the columns without NaN, which both passes compute: each within (u_P + 5e-4) sum p |v| + u_out |out| of the exact value
(tests/test_gpu_attention_prompt.py), and sum p |v| below 0.9 (0.80 for normal values).  Queries of the longest case are small, so that no
weight falls below f16's normal range whatever the number of positions."""
import math

import pytest
import torch

import leviathan_b200 as lev
from test_gpu_attention_prompt import U, Paged, i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def same_but_for_column_3(before, got):
    assert got[..., 3].isnan().all()
    got = got.clone()
    got[..., 3] = before[..., 3]
    assert before.isfinite().all() and got.isfinite().all()
    u = U[torch.float16]
    assert ((got - before).float().abs() <= 2 * ((u + 5e-4) * 0.9 + u * before.float().abs() + 1e-7)).all()


@pytest.mark.parametrize("heads,chunks,new", [((16, 8, 256), 16, 128), ((32, 8, 128), 24, 64)])
def test_more_units_than_find_room(ctx, heads, chunks, new):
    """pairs of CTAs; two tiles per CTA"""
    qh, kvh, hd = heads
    P = Paged([20000 + new], 16, kvh, hd, 5, spare=0)
    q = torch.randn((chunks * new, qh, hd), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).half()
    args = (i32([new * c for c in range(chunks + 1)]), i32([0] * chunks), i32([20000] * chunks), q, 0, hd ** -0.5)
    before = ctx.attn_chunk(P.cache, *args, dtype=torch.float16)
    P.v[int(P.table[0, 0]), 5, :, 3] = math.nan
    got = ctx.attn_chunk(P.cache, *args, dtype=torch.float16)
    ctx.synchronize()
    same_but_for_column_3(before, got)


def test_a_second_pass_of_twenty_seconds(ctx):
    """64 tokens behind POSITIONS positions among single tokens of other sequences, pages shared: the memory is small"""
    page, blocks, seqs, new = 16, 97, 296, 64
    need = (POSITIONS + new + page - 1) // page
    g = torch.Generator(device=DEV).manual_seed(5)
    k, v = (torch.randn((blocks, page, 1, 128), generator=g, device=DEV).half() for _ in range(2))
    table = torch.randint(1, blocks, (seqs, need), generator=g, device=DEV).to(torch.int32)
    table[0, 0] = 0   # the block of the NaN, in this place only
    rows = new + seqs - 1
    q = torch.randn((rows, 2, 128), generator=g, device=DEV).half() / 8
    starts = [0] + list(range(new, rows + 1))
    args = (i32(starts), i32(list(range(seqs))), i32([POSITIONS] + [s % 11 for s in range(1, seqs)]), q, 0, 128 ** -0.5)
    cache = lev.PagedKV.over(k, v, table)
    before = ctx.attn_chunk(cache, *args, dtype=torch.float16)
    v[0, 5, :, 3] = math.nan
    got = ctx.attn_chunk(cache, *args, dtype=torch.float16)
    ctx.synchronize()
    same_but_for_column_3(before[:new], got[:new])
    assert torch.equal(before[new:], got[new:])


POSITIONS = 300000
