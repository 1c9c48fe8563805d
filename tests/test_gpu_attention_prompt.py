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


@pytest.mark.parametrize("page", [1, 3, 5, 8, 16, 24, 32, 40, 48, 64, 96, 100, 128, 160, 256, 384])
@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128)])
def test_page_sizes(ctx, page, heads):
    run_chunk(ctx, [70, 3], [333, 150], page, heads, seed=page)
    run_chunk(ctx, [1, 200, 1, 1, 5, 300], [1200, 30, 700, 1, 128, 0], page, heads, seed=page)


@pytest.mark.parametrize("window", [1, 2, 100, 128, 129, 1000])
@pytest.mark.parametrize("heads", HEADS)
def test_windows(ctx, window, heads):
    run_chunk(ctx, [200, 1, 65], [700, 900, 0], 16, heads, window=window, seed=window)


@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128)])
def test_f32_cache(ctx, page, heads):
    run_chunk(ctx, [150, 2], [200, 31], page, heads, kv_type=torch.float32)
    run_chunk(ctx, [300, 2, 500], [500, 900, 0], page, heads, kv_type=torch.float32, window=333)


@pytest.mark.parametrize("scale", [0.0, -0.07, 1.0])
def test_scales(ctx, scale):
    run_chunk(ctx, [90], [200], 16, (8, 2, 128) if scale != 1.0 else (2, 2, 128), scale=scale if scale != 1.0 else 0.3, window=150)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n", [1, 4, 33])
def test_long_cache_is_split(ctx, heads, n):
    run_chunk(ctx, [n], [2900], 16, heads, seed=n)


@pytest.mark.parametrize("heads", [(14, 2, 128), (5, 1, 256), (16, 1, 128), (11, 1, 128), (16, 8, 256)])
@pytest.mark.parametrize("lens,ctxs,window,page", [([1], [1500], 0, 16), ([3, 70, 0, 19], [700, 1290, 5, 1], 0, 16), ([200], [1900], 0, 32),
                                                   ([40, 9], [2100, 300], 900, 16), ([17, 2], [1000, 1500], 0, 5), ([129], [3], 0, 16)])
def test_parts_of_uneven_tiles(ctx, heads, lens, ctxs, window, page):
    """few units, so that clusters share their positions: rows that no number of parts divides, parts that some units have none of"""
    run_chunk(ctx, lens, ctxs, page, heads, window, seed=sum(lens))


@pytest.mark.parametrize("heads", [(7, 1, 128), (3, 1, 256), (4, 2, 128)])
@pytest.mark.parametrize("lens", [[600], [90, 1, 300]])
def test_parts_of_prompts(ctx, heads, lens):
    run_prompt(ctx, lens, heads, torch.float16)


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


def test_a_prompt_of_9000(ctx):
    run_prompt(ctx, [9000], (2, 1, 128), torch.bfloat16)


# ---- values that nothing attends to, indices outside the layout ----
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,n,at,window,page", [((16, 8, 256), 70, 300, 0, 16), ((8, 2, 128), 5, 900, 0, 16), ((16, 8, 256), 700, 100, 200, 16),
                                                    ((8, 2, 128), 700, 130, 100, 16), ((8, 2, 128), 9, 40, 0, 7)])
def test_unattended_cache_may_hold_anything(ctx, junk, heads, n, at, window, page):
    """Positions behind the last row and in front of every window, pages no entry names: NaN and infinities there change nothing.  A NaN among
    the new tokens reaches the rows from its own on (as far as the window), and only those."""
    qh, kvh, hd = heads
    P = Paged([at + n], page, kvh, hd, 5)
    k, v = (t.clone() for t in P.rows(0, at + n))
    used = P.table[0, :P.need[0]].long()
    mark = torch.ones(P.k.shape[0], dtype=torch.bool, device=DEV)
    mark[used] = False
    for pool in (P.k, P.v):
        pool[mark] = junk
        e = int(P.table[0, (at + n - 1) // page])
        pool[e, (at + n - 1) % page + 1:] = junk          # behind the last position, in its page
        for p in range(max(0, at + 1 - window) if window else 0):
            pool[int(P.table[0, p // page]), p % page] = junk
    q = torch.randn((n, qh, hd), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    args = (i32([0, n]), i32([0]), i32([at]), q, window, hd ** -0.5)
    got = ctx.attn_chunk(P.cache, *args)
    ctx.synchronize()
    ref, mag = reference(q.half(), k, v, at, window, hd ** -0.5)
    check(got, ref, mag, torch.float16)
    first = n // 2
    pool_v = P.v[int(P.table[0, (at + first) // page])]
    pool_v[(at + first) % page, 0, 3] = junk
    got2 = ctx.attn_chunk(P.cache, *args)
    ctx.synchronize()
    g = qh // kvh
    last = min(n, first + window) if window else n
    hit = got2[first:last, :g, 3].float()
    assert (hit.isnan() if math.isnan(junk) else hit == junk).all()
    clean = torch.ones_like(got2, dtype=torch.bool)
    clean[first:last, :g, 3] = False
    assert got2[clean].isfinite().all()
    check(torch.where(clean, got2, got), ref, mag, torch.float16)


def test_nan_far_back_in_a_long_cache(ctx):
    """Every row attends to a NaN: its column is NaN, the others are what they were, and no wait runs out meanwhile (128 units of 128 rows
    that are all gone over again, about a second and a half)."""
    P = Paged([45064], 16, 8, 256, 5, spare=0)
    q = torch.randn((16 * 64, 16, 256), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).half()
    args = (i32([64 * c for c in range(17)]), i32([0] * 16), i32([45000] * 16), q, 0, 1 / 16)
    before = ctx.attn_chunk(P.cache, *args, dtype=torch.float16)
    P.v[int(P.table[0, 0]), 5, :, 3] = math.nan
    got = ctx.attn_chunk(P.cache, *args, dtype=torch.float16)
    ctx.synchronize()
    assert got[..., 3].isnan().all()
    got[..., 3] = before[..., 3]
    assert before.isfinite().all() and got.isfinite().all()
    # each is as close to the exact answer as `check` asks; the sum of p |v| over so many normal values is 0.80, below 0.9
    u = U[torch.float16]
    assert ((got - before).float().abs() <= 2 * ((u + 5e-4) * 0.9 + u * before.float().abs() + 1e-7)).all()


@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128), (32, 8, 128)])
@pytest.mark.parametrize("new,page", [(3, 16), (3, 128), (90, 64), (150, 128), (11, 24)])
def test_what_lies_behind_the_last_position_changes_no_bit(ctx, heads, new, page):
    """Sequences that end at every remainder of 16 (and with it of a step of 128), NaN against zeros behind each of them."""
    qh, kvh, hd = heads
    seqs = 33
    new_of = [new + s % 5 for s in range(seqs)]
    at = [s * 17 for s in range(seqs)]
    P = Paged([a + n for a, n in zip(at, new_of)], page, kvh, hd, 7)
    rows = [0]
    for n in new_of:
        rows.append(rows[-1] + n)
    q = torch.randn((rows[-1], qh, hd), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).half()
    outs = []
    for junk in (0.0, math.nan):
        for s in range(seqs):
            end = at[s] + new_of[s]
            for pool in (P.k, P.v):
                if end % page:
                    pool[int(P.table[s, end // page]), end % page:] = junk
        outs.append(ctx.attn_chunk(P.cache, i32(rows), i32(list(range(seqs))), i32(at), q, 0, hd ** -0.5))
        ctx.synchronize()
    assert outs[0].isfinite().all()
    assert torch.equal(*outs)


@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128), (32, 8, 128)])
@pytest.mark.parametrize("lens", [[1], [130, 15], [700], [40] * 37 + [129]])
def test_rows_behind_the_last_prompt_change_no_bit(ctx, heads, lens):
    qh, kvh, hd = heads
    rows = sum(lens)
    start = i32([sum(lens[:i]) for i in range(len(lens) + 1)])
    g = torch.Generator(device=DEV).manual_seed(9)
    outs = []
    q, k, v = (torch.randn((rows + 200, h, hd), generator=g, device=DEV).bfloat16() for h in (qh, kvh, kvh))
    for junk in (0.0, math.nan):
        for t in (q, k, v):
            t[rows:] = junk
        out = torch.full_like(q, 7.0)
        ctx.attn_prompt(q, k, v, start, 0, hd ** -0.5, out=out)
        ctx.synchronize()
        assert (out[rows:] == 7.0).all()
        outs.append(out[:rows])
    assert outs[0].isfinite().all()
    assert torch.equal(*outs)


@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128)])
def test_other_prompts_may_hold_anything(ctx, heads):
    qh, kvh, hd = heads
    g = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn((600, qh + 2 * kvh, hd), generator=g, device=DEV).to(torch.bfloat16)
    x[200:410] = math.nan
    q, k, v = x[:, :qh], x[:, qh:qh + kvh], x[:, qh + kvh:]
    got = ctx.attn_prompt(q, k, v, i32([0, 200, 410, 600]), 0, hd ** -0.5)
    ctx.synchronize()
    for a, b in ((0, 200), (410, 600)):
        ref, mag = reference(q[a:b], k[a:b], v[a:b], 0, 0, hd ** -0.5)
        check(got[a:b], ref, mag, torch.bfloat16)
    assert got[200:410].isnan().all()


@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("heads", [(16, 8, 256), (8, 2, 128)])
@pytest.mark.parametrize("kind", ["slot", "slot_negative", "pos", "pos_negative", "entry", "entry_negative"])
def test_bad_indices_are_reported_and_not_followed(ctx, heads, page, kind):
    qh, kvh, hd = heads
    lens, ctxs = [40, 300, 3], [200, 50, 77]
    P = Paged([a + b for a, b in zip(lens, ctxs)], page, kvh, hd, 9)
    slot, pos = [0, 1, 2], list(ctxs)
    if kind == "slot":
        slot[1] = 3
    elif kind == "slot_negative":
        slot[1] = -1
    elif kind == "pos":
        pos[1] = P.table.shape[1] * page - 299
    elif kind == "pos_negative":
        pos[1] = -1
    else:
        P.table[1, 2] = P.k.shape[0] if kind == "entry" else -1
    q = torch.randn((343, qh, hd), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    got = ctx.attn_chunk(P.cache, i32([0, 40, 340, 343]), i32(slot), i32(pos), q, 0, hd ** -0.5)
    with pytest.raises(lev.LevError, match="badDimensions"):
        ctx.synchronize()
    ctx.synchronize()   # reported once
    assert got[40:340].isnan().all()
    for c, (a, b) in ((0, (0, 40)), (2, (340, 343))):
        k, v = P.rows(c, lens[c] + ctxs[c])
        ref, mag = reference(q[a:b].half(), k, v, ctxs[c], 0, hd ** -0.5)
        check(got[a:b], ref, mag, torch.float16)


@pytest.mark.parametrize("starts", [[0, 9, 5, 20], [0, 9, 25, 20], [-1, 9, 9, 20], [0, 9, 9, 21]])
def test_bad_ranges_are_reported_and_left_out(ctx, starts):
    x = torch.randn((20, 4, 128), device=DEV).to(torch.float16)
    out = torch.full((20, 2, 128), 7.0, dtype=torch.float16, device=DEV)
    ctx.attn_prompt(x[:, :2], x[:, 2:3], x[:, 3:], i32(starts), out=out)
    with pytest.raises(lev.LevError, match="badDimensions"):
        ctx.synchronize()
    good = [(a, b) for a, b in zip(starts, starts[1:]) if 0 <= a <= b <= 20]
    for r in range(20):
        assert bool((out[r] == 7.0).all()) == (not any(a <= r < b for a, b in good)), r


def test_all_chunks_empty_or_rows_outside(ctx):
    out = torch.full((30, 2, 128), 7.0, dtype=torch.float16, device=DEV)
    x = torch.randn((30, 4, 128), device=DEV).to(torch.float16)
    ctx.attn_prompt(x[:, :2], x[:, 2:3], x[:, 3:], i32([5, 5, 5]), out=out)
    ctx.synchronize()
    assert (out == 7.0).all()
    ctx.attn_prompt(x[:, :2], x[:, 2:3], x[:, 3:], i32([5, 12]), out=out)
    ctx.synchronize()
    assert (out[:5] == 7.0).all() and (out[12:] == 7.0).all() and (out[5:12] != 7.0).any(-1).all()


@pytest.mark.parametrize("seqs", [33, 150, 1000])
def test_many_sequences(ctx, seqs):
    lens = [1 + (7 * i) % 13 for i in range(seqs)]
    run_prompt(ctx, lens, (8, 2, 128), torch.float16)


def test_output_rows_a_stride_apart(ctx):
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn((150, 6, 128), generator=g, device=DEV).to(torch.bfloat16)
    wide = torch.full((150, 7, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    got = ctx.attn_prompt(x[:, :4], x[:, 4:5], x[:, 5:], i32([0, 150]), 0, 0.1, out=wide[:, 1:5])
    ctx.synchronize()
    ref, mag = reference(x[:, :4], x[:, 4:5], x[:, 5:], 0, 0, 0.1)
    check(got, ref, mag, torch.bfloat16)
    assert (wide[:, 0] == 7.0).all() and (wide[:, 5:] == 7.0).all()


def test_long_offsets(ctx):
    """a pool of more than 2^32 bytes: rows of its last blocks"""
    hd, kvh, page = 256, 8, 64
    blocks = (5 << 30) // (page * kvh * hd * 2)
    k = torch.zeros((blocks, page, kvh, hd), dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator(device=DEV).manual_seed(1)
    table = i32([[blocks - 1, 3, blocks - 2, blocks - 9]])
    for e in table[0].tolist():
        k[e].normal_(generator=g)
        v[e].normal_(generator=g)
    q = torch.randn((20, 16, hd), generator=g, device=DEV)
    got = ctx.attn_chunk(lev.PagedKV.over(k, v, table), i32([0, 20]), i32([0]), i32([230]), q, 0, 1 / 16)
    ctx.synchronize()
    e = table[0].long()
    ref, mag = reference(q.half(), k[e].flatten(0, 1)[:250], v[e].flatten(0, 1)[:250], 230, 0, 1 / 16)
    check(got, ref, mag, torch.float16)


def test_repeats_captures_and_streams(ctx):
    """the same bits eager, captured and replayed, and from two contexts at once on two streams"""
    P = Paged([700, 1300], 16, 8, 256, 4)
    q = torch.randn((300, 16, 256), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    args = (i32([0, 100, 300]), i32([0, 1]), i32([600, 1100]), q, 0, 1 / 16)
    few = (i32([0, 2, 5]), i32([0, 1]), i32([690, 1290]), q[:5], 0, 1 / 16)   # merged over a cluster
    want, want_few = ctx.attn_chunk(P.cache, *args), ctx.attn_chunk(P.cache, *few)
    for _ in range(3):
        assert torch.equal(ctx.attn_chunk(P.cache, *args), want) and torch.equal(ctx.attn_chunk(P.cache, *few), want_few)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            a, b = ctx.attn_chunk(P.cache, *args), ctx.attn_chunk(P.cache, *few)
        a.zero_(), b.zero_()
        g.replay()
        g.replay()
    s.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want_few)
    other = lev.Context(0)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            outs.append((ctx.attn_chunk(P.cache, *args), want))
        with torch.cuda.stream(s2):
            outs.append((other.attn_chunk(P.cache, *few), want_few))
            outs.append((other.attn_chunk(P.cache, *args), want))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in outs)
    other.close()


def test_agrees_with_the_single_query_form(ctx):
    P = Paged([400], 16, 8, 256, 11)
    q = torch.randn((9, 16, 256), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    one = ctx.attn_decode(P.cache, i32([0] * 9), i32(list(range(391, 400))), q, 0, 1 / 16)
    got = ctx.attn_chunk(P.cache, i32([0, 9]), i32([0]), i32([391]), q, 0, 1 / 16, dtype=torch.float16)
    ctx.synchronize()
    # queries and weights rounded to f16 on one side only: 2^-11 of each score's terms and of each weight
    assert (got.float() - one).abs().max() <= 6e-3 * one.abs().max()


def test_refusals(ctx):
    P = Paged([64], 16, 2, 128, 1)
    st, sl, ps = i32([0, 8]), i32([0]), i32([5])
    q = torch.randn((8, 4, 128), device=DEV)
    half = q.half()
    ok = ctx.attn_chunk(P.cache, st, sl, ps, q)
    assert ok.dtype is torch.bfloat16
    for e, call in [(TypeError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q.to(torch.bfloat16))), (TypeError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q, out=q.clone())),
                    (ValueError, lambda: ctx.attn_chunk(P.cache, st.long(), sl, ps, q)), (ValueError, lambda: ctx.attn_chunk(P.cache, sl, sl, ps, q)),
                    (ValueError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q.transpose(0, 1))), (ValueError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q[..., :64])),
                    (ValueError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q.cpu())), (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q[:, :3].contiguous())),
                    (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q, window=-1)), (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, q, scale=math.inf)),
                    (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, torch.randn((8, 34, 128), device=DEV))),
                    (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, half, out=half)),
                    (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, torch.randn(8 * 512 + 1, device=DEV)[1:].view(8, 4, 128))),
                    (lev.LevError, lambda: ctx.attn_chunk(P.cache, st, sl, ps, torch.randn((8, 513), device=DEV)[:, :512].unflatten(1, (4, 128)))),
                    (TypeError, lambda: ctx.attn_prompt(half, half[:, :2], half[:, :2].to(torch.bfloat16), st)), (TypeError, lambda: ctx.attn_prompt(q, q[:, :2], q[:, :2], st)),
                    (ValueError, lambda: ctx.attn_prompt(half, half[:7, :2], half[:7, :2], st)), (lev.LevError, lambda: ctx.attn_prompt(half, half[:, :3], half[:, :3], st)),
                    (lev.LevError, lambda: ctx.attn_prompt(half[..., :64].contiguous(), half[:, :2, :64].contiguous(), half[:, :2, :64].contiguous(), st)),
                    (lev.LevError, lambda: ctx.attn_prompt(half, half[:, :2], half[:, 2:], st, out=half)),
                    (ValueError, lambda: lev.PagedKV.over(P.k, P.v[:, :8], P.table)), (TypeError, lambda: lev.PagedKV.over(P.k.to(torch.bfloat16), P.v.to(torch.bfloat16), P.table)),
                    (ValueError, lambda: lev.PagedKV.over(P.k, P.v, P.table.long()))]:
        with pytest.raises(e):
            call()
    ctx.synchronize()
