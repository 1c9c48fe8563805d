"""lev_norm_residual against its formula in 64 bits.

Tolerance.  Every output is a handful of f32 roundings (2^-24 each) of quantities of the size of |residual| + |alpha gate b|; a statistic is a
sum of n squares in f32 partial sums of at most n / 256 terms and a tree: (n / 256 + 13) 2^-24 relative, half of that after the root, so 1e-6
for n = 8192.  out: 2e-6 (|residual| + |alpha gate b|) |scale|; h: 4e-6 of the same times |inverse pre| plus its own rounding to 16 bits."""
import math

import pytest
import torch

import leviathan_b200 as lev

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def check(ctx, rows, n, norm_post=True, post=True, pre=True, gate=None, alpha=0.7, scale=1.3, dtype=torch.bfloat16, place=None, eps=1e-6, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + n)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    x, res = r(rows, n) * 0.5, r(rows, n) * 2
    w1, w2 = (1 + 0.1 * r(n) if norm_post and post else None), (1 + 0.1 * r(n) if pre else None)
    gt = {None: None, "row": r(n), "rows": r(rows, n), "strided": r(rows, n + 4)[:, :n]}[gate]
    b = x.double()
    if norm_post:
        b = b / torch.sqrt(b.square().mean(1, keepdim=True) + eps) * (w1.double() if w1 is not None else 1)
    add = alpha * (gt.double() if gt is not None else 1) * b
    want = scale * (res.double() + add)
    inv = 1 / torch.sqrt(want.square().mean(1, keepdim=True) + eps)
    p = w2.double() if w2 is not None else torch.ones(n, dtype=torch.float64, device=DEV)
    mag = abs(scale) * (res.double().abs() + add.abs())
    x0, res0 = x.clone(), res.clone()
    out, h = ctx.norm_residual(x, res, post=w1, pre=w2, gate=gt, alpha=alpha, scale=scale, eps=eps, norm_post=norm_post,
                               out={None: None, "x": x, "residual": res}[place], dtype=dtype)
    ctx.synchronize()
    assert ((out.double() - want).abs() <= 2e-6 * mag + 1e-12).all()
    wh = want * inv * p
    assert ((h.double() - wh).abs() <= 4e-6 * (mag * inv * p.abs()) + U[dtype] * wh.abs() * 1.001 + 1e-7).all()
    if place != "x":
        assert torch.equal(x, x0)
    if place != "residual":
        assert torch.equal(res, res0)
    only, none = ctx.norm_residual(x0, res0, post=w1, pre=w2, gate=gt, alpha=alpha, scale=scale, eps=eps, norm_post=norm_post, h=False)
    ctx.synchronize()
    assert none is None and torch.equal(only, out)


@pytest.mark.parametrize("n", [1, 3, 4, 255, 1024, 2816, 4096, 4097, 4100, 8192])
@pytest.mark.parametrize("rows", [1, 2, 67])
def test_sizes(ctx, rows, n):
    check(ctx, rows, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm_post,post,pre", [(False, False, True), (True, False, False), (True, True, True), (False, False, False)])
@pytest.mark.parametrize("n", [512, 513])
def test_forms(ctx, n, norm_post, post, pre, dtype):
    check(ctx, 5, n, norm_post, post, pre, dtype=dtype)


@pytest.mark.parametrize("gate", ["row", "rows", "strided"])
@pytest.mark.parametrize("n", [640, 641])
def test_gates(ctx, n, gate):
    check(ctx, 9, n, gate=gate)


@pytest.mark.parametrize("place", ["x", "residual"])
@pytest.mark.parametrize("n", [2816, 999, 5000])
def test_in_place(ctx, n, place):
    check(ctx, 4, n, place=place)


def test_zero_scales(ctx):
    check(ctx, 3, 256, alpha=0.0)
    check(ctx, 3, 256, scale=0.0)
    check(ctx, 3, 256, scale=-2.0, alpha=-1.0)


def test_equals_the_separate_calls(ctx):
    """residual sum, norm and bf16 conversion of the layer loop, one launch instead of three"""
    x, res, w = (torch.randn(s, device=DEV) for s in ((33, 2816), (33, 2816), (2816,)))
    out, h = ctx.norm_residual(x, res, pre=w, dtype=torch.bfloat16)
    ref = ctx.axpy(1.0, x, res)
    hb = ctx.act_bf16(ctx.rmsnorm(ref, w))
    ctx.synchronize()
    assert torch.equal(out, ref)
    # the sums of squares run in the same order; one product may round the other way before the 16-bit rounding
    assert ((h.float() - hb.float()).abs() <= 2 * U[torch.bfloat16] * hb.float().abs()).all() and (h != hb).float().mean() < 0.01


def test_refusals(ctx):
    x, res, w = torch.randn(4, 64, device=DEV), torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    flat = torch.zeros(5 * 64, device=DEV)
    for kw in (dict(out=flat[4:260].view(4, 64), x=flat[:256].view(4, 64)), dict(h=x), dict(h=res), dict(eps=-1.0), dict(alpha=math.inf), dict(scale=math.nan),
               dict(post=w, norm_post=False)):
        kw = dict(dict(x=x, residual=res, pre=w), **kw)
        with pytest.raises(lev.LevError):
            ctx.norm_residual(**kw)
    for kw in (dict(x=x.double()), dict(x=x.t()), dict(residual=res[:3]), dict(pre=w[:5]), dict(gate=torch.ones(3, device=DEV)), dict(h=x[:3].clone()), dict(x=x.cpu())):
        kw = dict(dict(x=x, residual=res, pre=w), **kw)
        with pytest.raises((ValueError, TypeError)):
            ctx.norm_residual(**kw)


@pytest.mark.parametrize("rows,n", [(1, 2816), (300, 2816), (5, 9001)])
def test_captured_replayed_and_on_another_stream(ctx, rows, n):
    x, res, w1, w2 = (torch.randn(s, device=DEV) for s in ((rows, n), (rows, n), (n,), (n,)))
    out, h = ctx.norm_residual(x, res, post=w1, pre=w2, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    out2, h2 = torch.zeros_like(out), torch.zeros_like(h)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        a, b = ctx.norm_residual(x, res, post=w1, pre=w2, dtype=torch.bfloat16)
        out2.copy_(a)
        h2.copy_(b)
    for _ in range(2):
        out2.zero_()
        h2.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, out) and torch.equal(h2, h)
    with torch.cuda.stream(s):
        a, b = ctx.norm_residual(x, res, post=w1, pre=w2, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    assert torch.equal(a, out) and torch.equal(b, h)


@pytest.mark.parametrize("rows,n", [(4, 64), (300, 9000)])
def test_outputs_over_a_weight_are_refused(ctx, rows, n):
    """other thread blocks read the weights while rows are written"""
    x, res = torch.randn(rows, n, device=DEV), torch.randn(rows, n, device=DEV)
    flat = torch.zeros((rows + 1) * n, device=DEV)
    out, w, after = flat[:rows * n].view(rows, n), flat[(rows - 1) * n:rows * n], flat[rows * n:]
    for kw in (dict(out=out, post=w), dict(out=out, pre=w), dict(h=out, post=w), dict(h=out, pre=w), dict(out=out, gate=w), dict(h=out, gate=w)):
        with pytest.raises(lev.LevError, match="overlaps"):
            ctx.norm_residual(x, res, **kw)
    ctx.norm_residual(x, res, post=after, pre=after, out=out)   # right behind it is another matter
    ctx.synchronize()
