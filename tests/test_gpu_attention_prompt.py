"""Attention of many rows per sequence (lev_attn_chunk over a paged cache, lev_attn_prompt over packed prompts) against the
formula in 64 bits.

Tolerance, element by element.  The reference takes the queries as the tensor core sees them (f32 queries rounded to f16), so what is
left is: the weights P rounded to 16 bits (half a step: 2^-11 for f16, 2^-8 for bf16) before the product with V, the output rounded to 16
bits, and f32 arithmetic.  With A = sum_j p_j |v_j| the first is at most u_P A.  Scores are f32 sums of 256 products: with standard
normal operands scale * sum |q k| is about 10, and 256 * 2^-24 * 10 = 1.5e-4 bounds their error, which changes a weight by twice that
(its own and the sum's).  Weights below 2^-14 lie on a grid of 2^-24 of a row's largest: n * 2^-25 <= 1e-4 for the 3000 positions here.
Together (u_P + 5e-4) A + u_out |out|."""
import math

import pytest
import torch

import leviathan_b200 as lev

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DEV = "cuda"


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def reference(q, k, v, first, window, scale):
    """q [m][heads][d] at positions first ..., k, v [n][kv heads][d] from position 0: (out, sum p |v|) in f64."""
    m, qh, d = q.shape
    g = qh // k.shape[1]
    out, mag = torch.empty((2, m, qh, d), dtype=torch.float64, device=q.device)
    p = first + torch.arange(m, device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)[None, :]
    allowed = (j <= p) & ((j > p - window) if window else torch.ones_like(j, dtype=torch.bool))
    for h in range(qh):
        kk, vv = k[:, h // g].double(), v[:, h // g].double()
        kk, vv = torch.nan_to_num(kk), torch.nan_to_num(vv)   # what is never attended to may be anything
        s = (q[:, h].double() @ kk.T) * scale
        w = torch.softmax(s.masked_fill(~allowed, -math.inf), -1)
        out[:, h], mag[:, h] = w @ vv, w @ vv.abs()
    return out, mag


def check(got, ref, mag, mma_type):
    tol = (U[mma_type] + 5e-4) * mag + U[got.dtype] * ref.abs() + 1e-7
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside: first {bad.nonzero()[0].tolist()}, worst {((got.double() - ref).abs() / tol).max():.3g} of the tolerance"


class Paged:
    """Sequences with a shuffled block table over pools that are filled behind every position."""

    def __init__(self, lens, page, kvh, hd, seed, dtype=torch.float16, spare=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        need = [(n + page - 1) // page for n in lens]
        blocks = sum(need) + spare
        order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
        self.table = torch.full((len(lens), max(need) + 1), -7, dtype=torch.int32, device=DEV)   # unused entries are no block
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at:at + m]
            at += m
        self.k = torch.randn((blocks, page, kvh, hd), generator=g, device=DEV).to(dtype)
        self.v = torch.randn((blocks, page, kvh, hd), generator=g, device=DEV).to(dtype)
        self.cache = lev.PagedKV.over(self.k, self.v, self.table)
        self.need = need

    def rows(self, s, n):
        e = self.table[s, :self.need[s]].long()
        return (self.k[e].flatten(0, 1)[:n], self.v[e].flatten(0, 1)[:n])


def run_chunk(ctx, lens, ctxs, page, heads, window=0, q_type=torch.float32, out_type=torch.bfloat16, kv_type=torch.float16, scale=None, seed=1,
              order=None, fused=True):
    qh, kvh, hd = heads
    scale = hd ** -0.5 if scale is None else scale
    P = Paged([a + b for a, b in zip(lens, ctxs)], page, kvh, hd, seed, kv_type)
    order = list(range(len(lens))) if order is None else order   # chunk c belongs to sequence order[c]
    rows = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    q = torch.randn((rows, qh + 2 * kvh if fused else qh, hd), generator=g, device=DEV).to(q_type)[:, :qh]
    starts = [0]
    for c in order:
        starts.append(starts[-1] + lens[c])
    out = torch.full((rows, qh, hd), 7.0, dtype=out_type, device=DEV)
    got = ctx.attn_chunk(P.cache, i32(starts), i32(order), i32([ctxs[c] for c in order]), q, window, scale, out=out)
    ctx.synchronize()
    for c, s in enumerate(order):
        a, b = starts[c], starts[c + 1]
        if a == b:
            continue
        k, v = P.rows(s, lens[s] + ctxs[s])
        ref, mag = reference(q[a:b].half(), k.half(), v.half(), ctxs[s], window, scale)
        check(got[a:b], ref, mag, torch.float16)


HEADS = [(16, 8, 256), (4, 4, 128), (8, 2, 128), (2, 2, 256)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n,at", [(1, 0), (2, 0), (5, 11), (128, 0), (129, 127), (300, 77)])
def test_one_chunk(ctx, heads, n, at):
    run_chunk(ctx, [n], [at], 16, heads, seed=n + at)


@pytest.mark.parametrize("heads", HEADS + [(14, 2, 128), (3, 1, 256), (16, 1, 128)])
@pytest.mark.parametrize("q_type,out_type", [(torch.float32, torch.bfloat16), (torch.float16, torch.float16)])
def test_several_sequences(ctx, heads, q_type, out_type):
    run_chunk(ctx, [1, 0, 37, 130, 64, 1, 257], [500, 3, 0, 1000, 63, 0, 129], 16, heads, q_type=q_type, out_type=out_type, order=[3, 0, 6, 1, 2, 5, 4])


@pytest.mark.parametrize("page", [1, 5, 8, 16, 24, 32, 64, 128, 256, 384])
@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128)])
def test_page_sizes(ctx, page, heads):
    run_chunk(ctx, [70, 3], [333, 150], page, heads, seed=page)


@pytest.mark.parametrize("window", [1, 2, 100, 128, 129, 1000])
@pytest.mark.parametrize("heads", HEADS)
def test_windows(ctx, window, heads):
    run_chunk(ctx, [200, 1, 65], [700, 900, 0], 16, heads, window=window, seed=window)


@pytest.mark.parametrize("page", [16, 7])
def test_f32_cache(ctx, page):
    run_chunk(ctx, [150, 2], [200, 31], page, (8, 2, 128), kv_type=torch.float32)


@pytest.mark.parametrize("scale", [0.0, -0.07, 1.0])
def test_scales(ctx, scale):
    run_chunk(ctx, [90], [200], 16, (8, 2, 128) if scale != 1.0 else (2, 2, 128), scale=scale if scale != 1.0 else 0.3, window=150)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n", [1, 4, 33])
def test_long_cache_is_split(ctx, heads, n):
    run_chunk(ctx, [n], [2900], 16, heads, seed=n)


@pytest.mark.parametrize("heads", HEADS)
def test_full_grid(ctx, heads):
    """enough tiles that nothing is split: CTA pairs, two tiles per CTA"""
    run_chunk(ctx, [1100, 901, 513], [200, 0, 1030], 16, heads, fused=False)


def run_prompt(ctx, lens, heads, dtype, window=0, seed=3, lead=0, tail=0):
    qh, kvh, hd = heads
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = lead + sum(lens) + tail
    fused = torch.randn((rows, qh + 2 * kvh, hd), generator=g, device=DEV).to(dtype)
    q, k, v = fused[:, :qh], fused[:, qh:qh + kvh], fused[:, qh + kvh:]
    starts = [lead]
    for n in lens:
        starts.append(starts[-1] + n)
    out = torch.full((rows, qh, hd), 7.0, dtype=dtype, device=DEV)
    got = ctx.attn_prompt(q, k, v, i32(starts), window, hd ** -0.5, out=out)
    ctx.synchronize()
    assert (got[:lead] == 7.0).all() and (got[rows - tail:] == 7.0).all()
    for a, b in zip(starts, starts[1:]):
        if b > a:
            ref, mag = reference(q[a:b], k[a:b], v[a:b], 0, window, hd ** -0.5)
            check(got[a:b], ref, mag, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS + [(14, 2, 128), (16, 1, 256)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 1], [128], [127, 1, 129, 300], [700, 513, 64, 1]])
def test_prompts(ctx, dtype, heads, lens):
    run_prompt(ctx, lens, heads, dtype, seed=len(lens), lead=3, tail=5)


@pytest.mark.parametrize("window", [1, 64, 129, 500])
@pytest.mark.parametrize("heads", HEADS)
def test_prompt_windows(ctx, window, heads):
    run_prompt(ctx, [640, 77], heads, torch.bfloat16, window=window)


@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128)])
def test_one_long_prompt(ctx, heads):
    run_prompt(ctx, [2500], heads, torch.bfloat16)
