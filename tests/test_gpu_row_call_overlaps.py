"""Outputs of the many-row calls over memory that other thread blocks still read are refused before anything is launched."""
import pytest
import torch

import leviathan_b200 as lev
from leviathan_b200 import _lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_over_its_own_cache(ctx, dtype):
    flat = torch.zeros(8 * 16 * 2 * 128 * 3, dtype=dtype, device=DEV)
    k, v, spare = (t.view(8, 16, 2, 128) for t in flat.chunk(3))
    table = i32([list(range(8))] * 300)
    q = torch.randn((8, 4, 128), device=DEV)
    cache = lev.PagedKV.over(k, v, table)
    args = (cache, i32([0, 8]), i32([0]), i32([20]), q)
    for pool in (k, v, table):
        out = pool.view(torch.float16).view(-1)[-8 * 512:].view(8, 4, 128)
        with pytest.raises(lev.LevError, match="overlaps the cache"):
            ctx.attn_chunk(*args, out=out)
    ctx.attn_chunk(*args, out=spare.view(torch.float16).view(-1)[:8 * 512].view(8, 4, 128))   # right behind the pools
    ctx.synchronize()


def test_scores_over_their_logits_or_one_another(ctx):
    rows, n, top = 40, 500, 3
    x = torch.zeros(rows * n + 4 * rows, device=DEV)
    after = [x[rows * n:][i * rows:(i + 1) * rows] for i in range(4)]
    tok, ids, lps = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(rows * top, dtype=torch.int32, device=DEV), torch.zeros(rows * top, device=DEV)

    def call(lp=after[0], ent=after[1], ids=ids, lps=lps, tokens=tok):
        p = lambda t: t.data_ptr()  # noqa: E731
        return L.load().lev_logprobs(ctx.handle, p(x), L.ELEM_F32, rows, n, n, 0.0, p(tokens), top, p(lp), p(ent), p(ids), p(lps))

    last = x[rows * n - 1:]
    for kw in (dict(lp=last), dict(ent=last), dict(ids=x), dict(lps=last), dict(lp=after[1]), dict(ids=lps), dict(lps=after[0]), dict(lp=tok), dict(ids=tok), dict(ent=tok)):
        assert L.STATUS[call(**kw)] == "badArgument", kw
    assert call() == L.OK
    ctx.synchronize()
