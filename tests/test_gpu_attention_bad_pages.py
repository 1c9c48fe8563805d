"""Pages outside the pool in a call of many units: each CTA (of a pair, both) goes from unit to unit, and only the rows of chunks that
attend to a bad page are NaN."""
import pytest
import torch

import leviathan_b200 as lev
from test_gpu_attention_prompt import Paged, check, i32, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("heads", [(16, 8, 256), (32, 8, 128), (16, 1, 128)])
@pytest.mark.parametrize("page", [16, 128, 20])
@pytest.mark.parametrize("new", [200, 40])
def test_bad_pages_among_many_units(heads, page, new):
    qh, kvh, hd = heads
    ctx = lev.Context(0)
    seqs = 60
    lens = [new + s % 7 for s in range(seqs)]
    at = [(s * 53) % 400 for s in range(seqs)]
    P = Paged([a + n for a, n in zip(at, lens)], page, kvh, hd, 4)
    bad = list(range(3, seqs, 5))
    page_of = {s: [0, P.need[s] - 1, P.need[s] // 2][s % 3] for s in bad}   # in turn the first page, the last one, one in between
    for s, e in page_of.items():
        P.table[s, e] = P.k.shape[0] + s if s % 2 else -1
    starts = [sum(lens[:i]) for i in range(seqs + 1)]
    q = torch.randn((starts[-1], qh, hd), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    for _ in range(3):
        got = ctx.attn_chunk(P.cache, i32(starts), i32(list(range(seqs))), i32(at), q, 0, hd ** -0.5)
        with pytest.raises(lev.LevError, match="badDimensions"):
            ctx.synchronize()
        for s in range(seqs):
            rows = got[starts[s]:starts[s + 1]]
            if s not in bad:
                assert rows.isfinite().all(), s
            else:   # rows in front of the page do not attend to it: theirs may be either
                assert rows[max(0, page_of[s] * page - at[s]):].isnan().all(), s
    for s in (0, 1, seqs - 1):
        k, v = P.rows(s, at[s] + lens[s])
        ref, mag = reference(q[starts[s]:starts[s + 1]], k, v, at[s], 0, hd ** -0.5)
        check(got[starts[s]:starts[s + 1]], ref, mag, torch.float16)
    ctx.close()
