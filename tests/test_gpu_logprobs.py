"""lev_logprobs against the definition in 64 bits: log probabilities of given tokens, entropy, top alternatives.

Tolerance.  x - lse and the entropy are sums of f32 quantities of the size of |x| + |lse| (below 100 here): a few roundings of 2^-24 of
that, the sum of weights (trees of f32 partial sums of at most 1200 terms, each weight off by the exponent's rounding, |x - m| log2(e)
2^-24 < 1e-5 relative where the weight counts): 2e-5 absolute on the logarithm.  With a cap, tanh from an exponential is off by
3 * 2^-23 of 1, times a cap of at most 50: 2e-5.  Together 5e-5 absolute.  Indices are exact: the order is that of the logits as given."""
import math

import pytest
import torch

import leviathan_b200 as lev

pytestmark = pytest.mark.gpu
DEV = "cuda"
ATOL = 5e-5


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def reference(logits, tokens, top, cap):
    raw = logits.double()
    x = cap * torch.tanh(raw / cap) if cap else raw
    lp = torch.log_softmax(x, -1)
    ent = -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(-1)
    order = torch.where(raw.isnan(), -math.inf, raw)
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, tokens.long()[:, None])[:, 0], ent, ids.to(torch.int32), lp.gather(1, ids)


def check(ctx, logits, top, cap, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    tokens = torch.randint(0, logits.shape[1], (logits.shape[0],), generator=g, device=DEV).to(torch.int32)
    lp, ent, ids, lps = ctx.logprobs(logits, tokens, top=top, softcap=cap)
    ctx.synchronize()
    rlp, rent, rids, rlps = reference(logits, tokens, top, cap)
    assert (lp.double() - rlp).abs().max() <= ATOL
    assert (ent.double() - rent).abs().max() <= ATOL
    if top:
        assert torch.equal(ids, rids)
        assert (lps.double() - rlps).abs().max() <= ATOL
    again = ctx.logprobs(logits, tokens, top=top, softcap=cap)
    ctx.synchronize()
    for a, b in zip((lp, ent, ids, lps), again):
        assert a is None or torch.equal(a, b)


def randn(shape, seed, dtype=torch.float32, sigma=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * sigma).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (1, 2, 2), (3, 5, 0), (2, 63, 64 - 1), (1, 4097, 5), (5, 32768, 20), (1, 262144, 64), (40, 50021, 8),
                                        (700, 1000, 3), (17, 100003, 33)])
def test_shapes(ctx, dtype, cap, rows, n, top):
    check(ctx, randn((rows, n), rows + n, dtype), top, cap)


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_a_stride_apart(ctx, dtype, offset):
    check(ctx, randn((6, 9001), 1, dtype)[:, offset:offset + 8990], 7, 30.0)


@pytest.mark.parametrize("n", [4096, 40000, 262144])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_orders_that_fill_the_buffer(ctx, n, top):
    """ascending rows (every value beats the ones before), descending ones, all values equal, few distinct values"""
    up = torch.arange(n, device=DEV, dtype=torch.float32) * (8.0 / n)
    rows = torch.stack([up, up.flip(0), torch.full_like(up, 1.5), (torch.arange(n, device=DEV) % 3).float(), torch.zeros_like(up)])
    rows[4, ::2] = -0.0   # ties with 0
    check(ctx, rows, top, 0.0)
    check(ctx, rows, top, 50.0)


@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_large_and_peaked(ctx, cap):
    x = randn((4, 30000), 2)
    x[0] += 40.0
    x[1, 777] = 60.0
    x[2] *= 0.0
    x[3] -= 45.0
    check(ctx, x, 4, cap)


def test_masked_logits(ctx):
    """-inf is probability 0; rows with NaN, +inf or nothing left have no distribution but keep their order"""
    x = randn((5, 20000), 3)
    x[0, 5:] = -math.inf
    x[1, ::2] = -math.inf
    x[2, 123] = math.nan
    x[3] = -math.inf
    x[4, 9] = math.inf
    tokens = torch.tensor([3, 1, 7, 0, 9], dtype=torch.int32, device=DEV)
    lp, ent, ids, lps = ctx.logprobs(x, tokens, top=8)
    ctx.synchronize()
    rlp, rent, rids, rlps = reference(x[:2], tokens[:2], 8, 0.0)
    assert (lp[:2].double() - rlp).abs().max() <= ATOL and (ent[:2].double() - rent).abs().max() <= ATOL
    assert torch.equal(ids[:2], rids)
    fin = rlps > -math.inf
    assert torch.equal(fin, lps[:2] > -math.inf) and (lps[:2].double() - rlps)[fin].abs().max() <= ATOL
    assert lp[2:].isnan().all() and ent[2:].isnan().all() and lps[2:].isnan().all()
    want = torch.sort(torch.where(x.isnan(), -math.inf, x), dim=1, descending=True, stable=True).indices[:, :8].to(torch.int32)
    assert torch.equal(ids[2], want[2]) and torch.equal(ids[4], want[4])
    assert torch.equal(ids[3], torch.arange(8, dtype=torch.int32, device=DEV))


def test_nan_comes_behind_everything(ctx):
    x = torch.full((1, 300), math.nan, device=DEV)
    x[0, 200] = -math.inf
    x[0, 7] = 1.0
    ids = ctx.logprobs(x, None, top=5)[2]
    ctx.synchronize()
    assert ids[0].tolist() == [7, 200, 0, 1, 2]


def test_given_tokens(ctx):
    x = randn((4, 5000), 4)
    tokens = torch.tensor([17, -1, 5000, -2], dtype=torch.int32, device=DEV)
    lp = ctx.logprobs(x, tokens)[0]
    with pytest.raises(lev.LevError, match="badDimensions"):
        ctx.synchronize()
    assert lp[1] == 0.0 and lp[2].isnan() and lp[3].isnan()
    assert abs(lp[0].item() - torch.log_softmax(x[0].double(), 0)[17].item()) <= ATOL
    ctx.synchronize()


def test_refusals(ctx):
    x = randn((2, 100), 5)
    tok = torch.zeros(2, dtype=torch.int32, device=DEV)
    for kw in (dict(top=65), dict(top=101), dict(top=-1), dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=math.nan)):
        with pytest.raises(lev.LevError):
            ctx.logprobs(x, tok, **kw)
    with pytest.raises(TypeError):
        ctx.logprobs(x.double(), tok)
    with pytest.raises(ValueError):
        ctx.logprobs(x, tok[:1])
    with pytest.raises(ValueError):
        ctx.logprobs(x, tok.long())
    with pytest.raises(ValueError):
        ctx.logprobs(x.t(), tok)
    with pytest.raises(ValueError):
        ctx.logprobs(x.cpu(), tok)


def test_captured_and_replayed(ctx):
    x, tok = randn((3, 40000), 6), torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    want = ctx.logprobs(x, tok, top=5, softcap=30.0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = ctx.logprobs(x, tok, top=5, softcap=30.0)
        g.replay()
        g.replay()
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
