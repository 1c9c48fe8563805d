"""lev_logprobs over masked vocabularies, against the definition in 64 bits: masks of -inf and of large finite values down to the type's lowest,
without a cap, over whole batches, threads, cluster parts, head and tail.

Tolerance: that of tests/test_gpu_logprobs.py, 5e-5 absolute (its derivation holds for live logits and log sums below 100; a masked logit far
below them has weight 0 in 64 bits too).  The log probability of a masked token itself is one f32 difference and two products on top of that:
2^-22 of its size."""
import math

import pytest
import torch

import leviathan_b200 as lev

pytestmark = pytest.mark.gpu
DEV = "cuda"
ATOL = 5e-5
MASKS = [-1e4, -65504.0, -1e9, -5e9, -1e10, -1e20, -1e30, -1e38, "lowest", -math.inf]


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def randn(shape, seed, sigma=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV) * sigma


def masked_rows(n, mask, centre=0.0, seed=0):
    """rows whose live places differ"""
    i = torch.arange(n, device=DEV)
    live = [i < n // 2, i >= n // 2, i % 2 == 1, (i // 16) % 2 == 1, (i // 1024) % 2 == 1, i == n - 1, i == 0, (i > n // 3) & (i < n // 3 + 20),
            i < 3, i >= n - 3, (i * 8 // n) % 2 == 1, i * 8 // n == 7, torch.ones_like(i, dtype=torch.bool)]
    x = randn((len(live), n), seed) + centre
    return torch.where(torch.stack(live), x, torch.full_like(x, mask))


def lowest(mask, dtype):
    return torch.finfo(dtype).min if mask == "lowest" else mask


def near(got, want):
    same = (got.double() == want) | (got.isnan() & want.isnan())
    ok = same | ((got.double() - want).abs() <= ATOL + 2.0 ** -22 * want.abs())
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off: {got[~ok][:4].tolist()} for {want[~ok][:4].tolist()}"


def check(ctx, x, cap, top):
    rows, n = x.shape
    raw = x.double()
    y = cap * torch.tanh(raw / cap) if cap else raw
    m = y.amax(1, keepdim=True)
    lp = (y - m) - torch.log(torch.exp(y - m).sum(1, keepdim=True))
    ent = -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(1)
    ids = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :top]
    for tokens in (raw.argmax(1), raw.argmin(1), torch.full((rows,), n - 1, device=DEV)):
        got, gent, gids, glps = ctx.logprobs(x, tokens.to(torch.int32), top=top, softcap=cap)
        ctx.synchronize()
        near(got, lp.gather(1, tokens[:, None])[:, 0])
        near(gent, ent)
        if top:
            assert torch.equal(gids.long(), ids)
            near(glps, lp.gather(1, ids))


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,top", [(2048, 0), (2048, 5), (40001, 3), (262144, 20)])
def test_masks_without_a_cap(ctx, n, top, dtype, mask):
    check(ctx, masked_rows(n, lowest(mask, dtype), seed=n).to(dtype), 0.0, top)


def test_f16_masks(ctx):
    for mask in (-65504.0, -math.inf):
        check(ctx, masked_rows(10007, mask).half(), 0.0, 4)


def nothing_but(ctx, rows, n, cap, mask):
    """every logit alike: -log n each, entropy log n; of -inf without a cap there is no distribution"""
    x = torch.full((rows, n), lowest(mask, torch.float32), device=DEV)
    lp, ent, ids, lps = ctx.logprobs(x, torch.full((rows,), n // 2, dtype=torch.int32, device=DEV), top=3, softcap=cap)
    ctx.synchronize()
    assert torch.equal(ids, torch.arange(3, dtype=torch.int32, device=DEV).expand(rows, 3))
    if mask == -math.inf and cap == 0.0:
        assert lp.isnan().all() and ent.isnan().all() and lps.isnan().all()
    else:
        for got, want in ((lp, -math.log(n)), (ent, math.log(n)), (lps, -math.log(n))):
            assert (got.double() - want).abs().max() <= ATOL


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("rows,n", [(1, 300), (1, 262144), (700, 5000)])
def test_rows_of_nothing_but_the_mask(ctx, rows, n, mask):
    nothing_but(ctx, rows, n, 0.0, mask)


@pytest.mark.parametrize("scale", [1e3, 1e5, 1e10, 1e30, 1e38])
@pytest.mark.parametrize("n", [2048, 40001])
def test_logits_of_any_size(ctx, n, scale):
    x = (randn((5, n), 8, 1.0) * scale).clamp(-3.4e38, 3.4e38)
    x[1] = x[1].abs()
    x[2] = -x[2].abs()
    x[3, :n // 2] = torch.finfo(torch.float32).min
    raw = x.double()
    lp = torch.log_softmax(raw, 1)
    ent = -torch.where(lp.exp() > 0, lp.exp() * lp, 0.0).sum(1)
    tokens = raw.argmax(1)
    got, gent, gids, glps = ctx.logprobs(x, tokens.to(torch.int32), top=4)
    ctx.synchronize()
    # the largest logits: differences of f32 numbers, exact to 2^-24 of the difference
    near(got, lp.gather(1, tokens[:, None])[:, 0])
    near(gent, ent)
    ids = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(gids.long(), ids)
    near(glps, lp.gather(1, ids))
