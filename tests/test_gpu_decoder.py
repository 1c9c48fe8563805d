"""The ends of a decode step (lev_embed_rows, lev_softcap) and the whole synthetic decoder step, eager and as
one CUDA graph, against the f64 oracle."""
import math

import numpy as np
import pytest
import torch

import leviathan_b200 as lev
from leviathan_b200 import quant as Q
from leviathan_b200.decoder import DecoderConfig, SyntheticDecoder
from oracle import oracle as O

from helpers import quantized, random_blocks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = lev.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("name,t,cols", [("q6_k", Q.GGML_Q6_K, 2816), ("q4_k", Q.GGML_Q4_K, 512), ("q4_0", Q.GGML_Q4_0, 96)])
@pytest.mark.parametrize("encoded", [True, False])
def test_embedding_rows_are_bit_exact(ctx, name, t, cols, encoded):
    rows = 40
    w = quantized(t, 11, rows, cols) if encoded else random_blocks(t, 12, rows, cols)
    wd = ctx.upload(torch.from_numpy(w).cuda(), t, rows, cols)
    toks = [0, 39, 17, 17, 3]
    scale = math.sqrt(cols)
    got = ctx.embed_rows(wd, torch.tensor(toks, dtype=torch.int32, device="cuda"), scale).cpu().numpy()
    for i, tk in enumerate(toks):
        want = O.embed_row(t, w, rows, cols, tk, scale)
        assert np.array_equal(got[i].view(np.uint32), want.view(np.uint32)), (name, tk)
    wd.free()


def test_embedding_row_outside_the_tensor_is_reported_not_read(ctx):
    w = quantized(Q.GGML_Q6_K, 5, 8, 256)
    wd = ctx.upload(torch.from_numpy(w).cuda(), Q.GGML_Q6_K, 8, 256)
    out = ctx.embed_rows(wd, torch.tensor([2, 8, -1], dtype=torch.int32, device="cuda"), 1.0)
    with pytest.raises(lev.LevError):
        ctx.synchronize()
    o = out.cpu().numpy()
    assert np.array_equal(o[0], O.embed_row(Q.GGML_Q6_K, w, 8, 256, 2, 1.0)) and not o[1].any() and not o[2].any()
    ctx.synchronize()  # the report was consumed
    wd.release_gguf()
    with pytest.raises(lev.LevError):
        ctx.embed_rows(wd, torch.tensor([1], dtype=torch.int32, device="cuda"), 1.0)
    wd.free()


def test_softcap(ctx):
    x = np.concatenate([Q.normal(3, (100000,), 20.0), np.array([0.0, -0.0, 1e-30, 1e4, -1e4, 88.0, -3e38, 3e38], np.float32)])
    got = ctx.softcap(torch.from_numpy(x.copy()).cuda(), 30.0).cpu().numpy()
    want = O.softcap_f64(x, 30.0)
    assert np.isfinite(got).all()
    assert np.max(np.abs(got - want) / np.maximum(1.0, np.abs(want))) < 4e-6
    assert np.array_equal(np.signbit(got), np.signbit(x))
    assert got[-1] == 30.0 and got[-2] == -30.0
    with pytest.raises(lev.LevError):
        ctx.softcap(torch.zeros(4, device="cuda"), 0.0)


SMALL = dict(hidden=256, layers=2, q_heads=4, kv_heads=2, head_dim=128, experts=8, top_k=2, expert_inter=64, vocab=512,
             positions=48, page=16)


def _reference_step(dec, cfg, batch, pos):
    """per sequence: the oracle's step over host copies of this decoder's tensors and caches"""
    out = []
    for s in range(batch):
        kc, vc = [], []
        for L in dec.layers:
            tab = L.cache.table_host[s]
            k = L.cache.k.cpu().numpy().reshape(-1, cfg.page, cfg.kv_heads, cfg.head_dim)
            v = L.cache.v.cpu().numpy().reshape(-1, cfg.page, cfg.kv_heads, cfg.head_dim)
            kc.append(np.concatenate([k[b] for b in tab])[:cfg.positions].copy())
            vc.append(np.concatenate([v[b] for b in tab])[:cfg.positions].copy())
        out.append(O.decode_step_f64(cfg, dec.host, int(dec.tok[s].item()), pos, kc, vc))
    return out


@pytest.mark.parametrize("batch", [1, 3, 11, 20])
def test_decoder_step_against_the_f64_oracle_eager_and_as_one_graph(ctx, batch):
    cfg = DecoderConfig(**SMALL)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        dec = SyntheticDecoder(ctx, cfg, batch=batch, keep_host_copies=True)
        dec.tok.copy_(torch.tensor([(7 * s + 5) % cfg.vocab for s in range(batch)], dtype=torch.int32))
        tok0 = dec.tok.clone()
        stream.synchronize()
        refs = _reference_step(dec, cfg, batch, cfg.positions - 1)
        dec.step()
        ctx.synchronize()
        logits = dec.logits.cpu().numpy().copy()
        toks = dec.tok.cpu().numpy().copy()
        for s in range(batch):
            want = refs[s]["logits"]
            err = np.max(np.abs(logits[s] - want)) / max(1.0, float(np.max(np.abs(want))))
            # from 16 sequences on the projections run on the tensor cores with bf16 activations (bar 2e-2)
            assert err < (2e-2 if dec.wide else 2e-4), (s, err)
            top2 = np.sort(want)[-2:]
            if top2[1] - top2[0] > (0.5 if dec.wide else 1e-3):
                assert toks[s] == refs[s]["token"]
            assert toks[s] == int(np.argmax(logits[s]))
        # the same step as one graph: same bits, and the token it leaves is the next step's input
        dec.tok.copy_(tok0)
        dec.capture()
        l0 = ctx.launch_count()
        dec.replay()
        ctx.synchronize()
        assert ctx.launch_count() == l0  # a replay makes no call into the library
        assert np.array_equal(dec.logits.cpu().numpy().view(np.uint32), logits.view(np.uint32))
        assert np.array_equal(dec.tok.cpu().numpy(), toks)
        dec.replay()
        ctx.synchronize()
        second = dec.tok.cpu().numpy().copy()
        dec.tok.copy_(torch.from_numpy(toks))
        dec.step()
        ctx.synchronize()
        assert np.array_equal(dec.tok.cpu().numpy(), second)
        dec.free()


# ---- prompts: the operators together, as a serving loop runs them ----
PROMPT = dict(SMALL, top_k=8, positions=176)   # every expert takes part: no near-tie of the router falls the other way


def _walk(dec, cfg, tokens):
    """the oracle's steps over a prompt from an empty cache: one dict per token"""
    kc = [np.zeros((cfg.positions, cfg.kv_heads, cfg.head_dim), np.float16) for _ in dec.layers]
    vc = [np.zeros_like(k) for k in kc]
    return [O.decode_step_f64(cfg, dec.host, int(t), p, kc, vc) for p, t in enumerate(tokens)]


def _near(got, want):
    # projections and experts' inputs in bf16, as in a wide decode step: the same bar
    err = np.max(np.abs(got - want)) / max(1.0, float(np.max(np.abs(want))))
    assert err < 2e-2, err


@pytest.mark.parametrize("batch", [2, 17])
def test_prompt_pieces_and_decode_steps_against_the_f64_oracle(ctx, batch):
    """two prompts taken in by pieces (one whole, one in three pieces, pieces of both in one call), then a decode step on top"""
    cfg = DecoderConfig(**PROMPT)
    dec = SyntheticDecoder(ctx, cfg, batch=batch, keep_host_copies=True, prompts=True)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.vocab, 23), rng.integers(0, cfg.vocab, 61)]
    refs = [_walk(dec, cfg, p) for p in prompts]
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    pieces = [[(1, 0, 20)], [(0, 0, 23), (1, 20, 59)], [(1, 59, 61)]]   # (sequence, from, to) of each call
    for call in pieces:
        toks = np.concatenate([prompts[s][a:b] for s, a, b in call])
        start = np.concatenate([[0], np.cumsum([b - a for _, a, b in call])])
        nxt, logits = dec.prefill(i32(toks), i32(start), i32([s for s, _, _ in call]), i32([a for _, a, _ in call]))
        ctx.synchronize()
        for i, (s, a, b) in enumerate(call):
            _near(logits[i].cpu().numpy(), refs[s][b - 1]["logits"])
            assert int(nxt[i]) == int(torch.argmax(logits[i]))
    # a decode step continues both sequences from the caches that the prompts left
    dec.tok[:2] = i32([5, 9])
    dec.pos[:2] = i32([23, 61])
    want = [_walk(dec, cfg, list(prompts[s]) + [t])[-1]["logits"] for s, t in ((0, 5), (1, 9))]
    dec.step()
    ctx.synchronize()
    for s in range(2):
        _near(dec.logits[s].cpu().numpy(), want[s])
    dec.free()


def test_scored_prompts_against_the_f64_oracle(ctx):
    cfg = DecoderConfig(**PROMPT)
    dec = SyntheticDecoder(ctx, cfg, batch=1, keep_host_copies=True, prompts=True)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, cfg.vocab, n) for n in (1, 37, 18)]
    toks = torch.tensor(np.concatenate(prompts), dtype=torch.int32, device="cuda")
    start = torch.tensor(np.concatenate([[0], np.cumsum([len(p) for p in prompts])]), dtype=torch.int32, device="cuda")
    lp, ent, ids, lps = dec.score(toks, start, top=3, rows=40)
    ctx.synchronize()
    row = 0
    for p in prompts:
        for i, r in enumerate(_walk(dec, cfg, p)):
            want = torch.log_softmax(torch.from_numpy(r["logits"]), 0)
            # a log probability moves by at most twice what the logits are off by (2e-2 of the largest)
            tol = 2 * 2e-2 * max(1.0, float(np.max(np.abs(r["logits"]))))
            if i + 1 < len(p):
                assert abs(float(lp[row]) - float(want[int(p[i + 1])])) <= tol
            else:
                assert float(lp[row]) == 0.0
            assert torch.all((lps[row].cpu() - want[ids[row].cpu().long()]).abs() <= tol)
            assert abs(float(ent[row]) + float((want.exp() * want).sum())) <= 2 * tol * float(want.abs().max())
            row += 1
    # the same rows through the caches: log probabilities of the last rows agree
    _, logits = dec.prefill(toks[1:38], torch.tensor([0, 37], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                            torch.zeros(1, dtype=torch.int32, device="cuda"))
    again = ctx.logprobs(logits, None, top=3)
    ctx.synchronize()
    # f16 cache and queries on one side, bf16 on the other: 2^-8 of a logit's size through two layers
    assert (again[3][0] - lps[37]).abs().max() <= 4e-2 * max(1.0, float(logits.abs().max()))
    dec.free()


def test_prompts_are_refused_without_their_tensors(ctx):
    dec = SyntheticDecoder(ctx, DecoderConfig(**SMALL), batch=1)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="prompts=True"):
        dec.prefill(one, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), one, one)
    dec.free()


def test_padding_of_a_prompt_batch_reaches_no_sequence(ctx):
    """a batch of fixed size: tokens in front of the first chunk and behind the last one are junk, and the caches keep what they held"""
    cfg = DecoderConfig(**PROMPT)
    dec = SyntheticDecoder(ctx, cfg, batch=3, prompts=True)
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    rng = np.random.default_rng(5)
    toks = rng.integers(0, cfg.vocab, 30)
    slot, pos = i32([2, 0]), i32([40, 7])
    pools = [t.clone() for L in dec.layers for t in (L.cache.k, L.cache.v)]
    want, logits = dec.prefill(i32(toks), i32([0, 11, 30]), slot, pos)
    ctx.synchronize()
    filled = [t.clone() for L in dec.layers for t in (L.cache.k, L.cache.v)]
    for t, p in zip((t for L in dec.layers for t in (L.cache.k, L.cache.v)), pools):
        t.copy_(p)
    padded = np.concatenate([[-1, 5, cfg.vocab, 1 << 30, 3], toks, [-7] * 9, rng.integers(0, cfg.vocab, 40)])
    got, padded_logits = dec.prefill(i32(padded), i32([5, 16, 35]), slot, pos)
    ctx.synchronize()
    _near(padded_logits.cpu().numpy(), logits.cpu().numpy())
    mine = {0: range(7, 26), 2: range(40, 51)}
    held = torch.ones(dec.layers[0].cache.k.shape[:2], dtype=torch.bool, device="cuda")
    held[0] = False   # the scratch block
    for s, positions in mine.items():
        for p in positions:
            held[dec.layers[0].cache.owned[s][p // cfg.page], p % cfg.page] = False
    for t, before, after in zip((t for L in dec.layers for t in (L.cache.k, L.cache.v)), pools, filled):
        assert torch.equal(t[held], before[held])
        _near(t[~held].float().cpu().numpy()[cfg.page:], after[~held].float().cpu().numpy()[cfg.page:])
    # a slot that is no sequence's is reported
    dec.prefill(i32(toks), i32([0, 11, 30]), i32([3, 0]), pos)
    with pytest.raises(lev.LevError, match="badDimensions"):
        ctx.synchronize()
    dec.free()


def test_padding_of_scored_prompts(ctx):
    cfg = DecoderConfig(**PROMPT)
    dec = SyntheticDecoder(ctx, cfg, batch=1, prompts=True)
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    rng = np.random.default_rng(6)
    toks = rng.integers(0, cfg.vocab, 40)
    lp, ent, ids, lps = dec.score(i32(toks), i32([0, 0, 15, 15, 40]), top=3)
    padded = np.concatenate([[-5, cfg.vocab], toks, [1 << 29] * 7])
    plp, pent, pids, plps = dec.score(i32(padded), i32([2, 2, 17, 17, 42]), top=3)
    ctx.synchronize()
    assert lp[14] == 0 and lp[39] == 0 and (lp[:14] < 0).all() and (lp[15:39] < 0).all()
    assert (plp[:2] == 0).all() and (plp[42:] == 0).all()
    for a, b in ((plp, lp), (pent, ent), (plps, lps)):
        _near(a[2:42].cpu().numpy(), b.cpu().numpy())
    dec.free()
