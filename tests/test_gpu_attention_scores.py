"""Attention of many rows per sequence at scores of any size, against the formula in 64 bits.  The scores here are exact in f32 (one product,
or a product and a small number), so the tolerance is that of tests/test_gpu_attention_prompt.py, (u_P + 5e-4) sum p |v| + u_out |out|."""
import pytest
import torch

import leviathan_b200 as lev
from test_gpu_attention_prompt import Paged, check, i32, reference

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


@pytest.mark.parametrize("size", [1e3, 2e9, 4e9])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n,at", [(5, 900), (200, 300), (1000, 0)])
def test_large_scores_over_the_cache(ctx, heads, n, at, sign, size):
    """one coordinate makes the score: the largest wins, equal ones share"""
    qh, kvh, hd = heads
    P = Paged([at + n], 16, kvh, hd, 3)
    a = min(65504.0, size ** 0.5)
    levels = torch.tensor([1.0, 0.5, 0.98, 0.25, 1.0, 0.99], device=DEV) * (size / a)
    q = torch.zeros((n, qh, hd), device=DEV)
    q[..., 0] = sign * a
    P.k[...] = 0.0
    P.k[..., 0] = levels[torch.randint(0, 6, P.k.shape[:3], generator=gen(5), device=DEV)].half()
    got = ctx.attn_chunk(P.cache, i32([0, n]), i32([0]), i32([at]), q, 0, 1.0)
    ctx.synchronize()
    k, v = P.rows(0, at + n)
    ref, mag = reference(q.half(), k, v, at, 0, 1.0)
    check(got, ref, mag, torch.float16)


@pytest.mark.parametrize("size", [1e12, 1e30])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens,window", [([700], 0), ([90, 3, 300], 50), ([2300], 0)])
def test_large_scores_of_prompts(ctx, heads, lens, window, size):
    qh, kvh, hd = heads
    rows = sum(lens)
    q, k = torch.zeros((rows, qh, hd), device=DEV), torch.zeros((rows, kvh, hd), device=DEV)
    q[..., 0] = size ** 0.5
    k[..., 0] = torch.tensor([1.0, 0.5, 1.0, 0.25, 0.75], device=DEV)[torch.randint(0, 5, (rows, kvh), generator=gen(2), device=DEV)] * size ** 0.5
    q, k, v = q.bfloat16(), k.bfloat16(), torch.randn((rows, kvh, hd), generator=gen(3), device=DEV).bfloat16()
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    got = ctx.attn_prompt(q, k, v, i32(starts), window, 1.0)
    ctx.synchronize()
    for a, b in zip(starts, starts[1:]):
        ref, mag = reference(q[a:b], k[a:b], v[a:b], 0, window, 1.0)
        check(got[a:b], ref, mag, torch.bfloat16)


@pytest.mark.parametrize("base", [0.0, 2.0 ** 12, 2.0 ** 15, -(2.0 ** 15)])
@pytest.mark.parametrize("heads", HEADS)
def test_scores_that_share_a_large_part(ctx, heads, base):
    """scores base * 16 + c, exact in f32: the weights depend on c alone.  c rises now and then, so that a row's reference moves while what
    lies behind it still counts."""
    qh, kvh, hd = heads
    n, at = 150, 1300
    P = Paged([at + n], 16, kvh, hd, 3)
    q = torch.zeros((n, qh, hd), device=DEV)
    q[..., 0], q[..., 1] = 16.0, 1.0
    p = torch.arange(at + n, device=DEV)
    c = (torch.randint(0, 16, (at + n,), generator=gen(6), device=DEV) / 16 + 6.0 * (p > 450) + 7.0 * (p > 1270)).half()
    e = P.table[0, p // 16].long()
    P.k[...] = 0.0
    P.k[e, p % 16, :, 0] = base
    P.k[e, p % 16, :, 1] = c[:, None]
    got = ctx.attn_chunk(P.cache, i32([0, n]), i32([0]), i32([at]), q, 0, 1.0)
    ctx.synchronize()
    k, v = P.rows(0, at + n)
    ref, mag = reference(q.half(), k, v, at, 0, 1.0)
    check(got, ref, mag, torch.float16)


@pytest.mark.parametrize("heads", HEADS)
def test_a_scale_of_zero_weighs_large_scores_alike(ctx, heads):
    qh, kvh, hd = heads
    q, k, v = (torch.randn((300, h, hd), generator=gen(h), device=DEV).bfloat16() for h in (qh, kvh, kvh))
    q[..., 0] = 1e17
    k[..., 0] *= 1e17
    got = ctx.attn_prompt(q, k, v, i32([0, 300]), 0, 0.0)
    ctx.synchronize()
    ref, mag = reference(q, k, v, 0, 0, 0.0)
    check(got, ref, mag, torch.bfloat16)
