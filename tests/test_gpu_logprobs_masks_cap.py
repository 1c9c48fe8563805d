"""lev_logprobs with a softcap over masked vocabularies, against the definition in 64 bits: there the value of -inf is -cap, whose weight is
not 0, and that of +inf the cap.  Tolerances and masked places: tests/test_gpu_logprobs_masks.py."""
import math

import pytest
import torch

import leviathan_b200 as lev
from test_gpu_logprobs_masks import MASKS, check, lowest, masked_rows, nothing_but, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("mask", [-1e4, -1e10, "lowest", -math.inf])
@pytest.mark.parametrize("centre", [0.0, -40.0, 30.0])
@pytest.mark.parametrize("cap", [1.0, 5.0, 10.0, 30.0])
@pytest.mark.parametrize("n,top", [(2048, 5), (40001, 3)])
def test_masks_under_a_cap(ctx, n, top, cap, centre, mask):
    x = masked_rows(n, lowest(mask, torch.float32), centre, seed=n + 1)
    check(ctx, x, cap, top)
    check(ctx, x[:, 1:n - 2], cap, top)   # head and tail that are no whole 16-byte units


@pytest.mark.parametrize("mask", [-65504.0, -math.inf])
def test_f16_masks_under_a_cap(ctx, mask):
    check(ctx, masked_rows(10007, mask).half(), 5.0, 4)


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("cap", [1.0, 30.0])
@pytest.mark.parametrize("rows,n", [(1, 300), (1, 262144), (700, 5000)])
def test_rows_of_nothing_but_the_mask_under_a_cap(ctx, rows, n, cap, mask):
    nothing_but(ctx, rows, n, cap, mask)


@pytest.mark.parametrize("cap", [1.0, 5.0, 30.0])
def test_infinities_under_a_cap(ctx, cap):
    """cap * tanh(inf / cap) is the cap: a distribution like any other; NaN leaves none"""
    x = randn((4, 3000), 3)
    x[0, 17] = math.inf
    x[1, 5:90] = math.inf
    x[2, 100:] = -math.inf
    check(ctx, x[:3], cap, 6)
    x[3, 2999] = math.nan
    lp, ent, ids, lps = ctx.logprobs(x, torch.zeros(4, dtype=torch.int32, device=DEV), top=6, softcap=cap)
    ctx.synchronize()
    assert lp[3].isnan() and ent[3].isnan() and lps[3].isnan().all() and not lp[:3].isnan().any()
