"""Attention of many rows per sequence: places that a row does not attend to have weight 0, whatever finite value lies there (outputs are
compared bit by bit), and a row without any weight has no value."""
import math

import pytest
import torch

import leviathan_b200 as lev
from test_gpu_attention_prompt import i32

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS = [(16, 8, 256), (4, 4, 128), (8, 2, 128), (2, 2, 256), (32, 8, 128)]


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("large", [2.0 ** 118, -(2.0 ** 120), 3e38])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens,window", [([300], 0), ([1100], 0), ([129, 200, 77], 0), ([700], 100), ([40] * 37 + [129], 0), ([2500], 900)])
def test_unattended_large_values_change_no_bit(ctx, heads, lens, window, large):
    """above the diagonal, in front of a window, in other prompts' rows"""
    qh, kvh, hd = heads
    rows, g = sum(lens), gen(len(lens))
    q, k, v = (torch.randn((rows, h, hd), generator=g, device=DEV).bfloat16() for h in (qh, kvh, kvh))
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    cut = lens[0] * 2 // 3           # rows 0 ... cut - 1 do not attend to the places from cut on
    after = cut + window if window else rows   # ... nor rows from `after` on to those before `cut + 1`
    outs = []
    for other in (0.0, large):
        w = v.clone()
        w[cut:] = other
        a = ctx.attn_prompt(q, k, w, i32(starts), window, hd ** -0.5)[:cut]
        w = v.clone()
        w[:cut + 1] = other
        b = ctx.attn_prompt(q, k, w, i32(starts), window, hd ** -0.5)
        ctx.synchronize()
        outs.append((a, b[after:lens[0]], b[lens[0]:]))
    for x, y in zip(*outs):
        assert x.isfinite().all() and torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("rows", [3, 700])
def test_rows_whose_scores_are_all_minus_infinity(ctx, heads, rows, dtype):
    """the formula has no value there; the next row attends to one finite score and takes its V"""
    qh, kvh, hd = heads
    q, k, v = (torch.randn((rows, h, hd), generator=gen(h), device=DEV).to(dtype) for h in (qh, kvh, kvh))
    q[:2] = 1.0
    k[0] = -math.inf
    q[2:, :, 0], q[2:, :, 1:] = 1.0, 0.0   # rows behind: -inf at the first place (0 times an infinity elsewhere would be NaN)
    k[0, :, 1:] = 0.0
    out = ctx.attn_prompt(q, k, v, i32([0, rows]), 0, hd ** -0.5)
    ctx.synchronize()
    assert out[0].isnan().all()
    assert torch.equal(out[1], v[1].repeat_interleave(qh // kvh, 0))
    assert out[1:].isfinite().all()
