"""The operators of prompt ingestion and scoring, as a host of this package calls them, with their plain forms.

  chunk     Context.attn_chunk: attention of a chunk of new tokens per sequence over a paged cache
  prompt    Context.attn_prompt: causal attention of whole prompts packed behind one another
  logprobs  Context.logprobs: log probability of given tokens, entropy and top alternatives of rows of logits
  norm      Context.norm_residual: norm behind a block, gate, residual sum and scale, norm before the next block
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # five drafted tokens of one sequence checked in one pass at a context of 4096
        dict(name="chunk_verify_5", kind="chunk", q_heads=16, kv_heads=8, head_dim=256, seqs=1, new_min=5, new_max=5,
             ctx_min=4091, ctx_max=4091, page=16, window=0, q="f32", out="bf16"),
        # the last piece of a long prompt that is taken in by pieces of 512 tokens
        dict(name="chunk_512_at_7680", kind="chunk", q_heads=16, kv_heads=8, head_dim=256, seqs=1, new_min=512, new_max=512,
             ctx_min=7680, ctx_max=7680, page=16, window=0, q="f32", out="bf16"),
        # prompt pieces and decoding sequences of a server in one call, lengths from 1 to 300, odd contexts
        dict(name="chunk_mixed_24", kind="chunk", q_heads=32, kv_heads=8, head_dim=128, seqs=24, new_min=1, new_max=300,
             ctx_min=37, ctx_max=4000, page=16, window=0, q="f16", out="f16"),
        # a layer with a sliding window, pages of another size
        dict(name="chunk_window", kind="chunk", q_heads=16, kv_heads=8, head_dim=256, seqs=3, new_min=400, new_max=701,
             ctx_min=0, ctx_max=3001, page=32, window=1024, q="f32", out="bf16"),
        # one prompt scored whole
        dict(name="prompt_4096", kind="prompt", q_heads=16, kv_heads=8, head_dim=256, seqs=1, len_min=4096, len_max=4096,
             window=0, type="bf16"),
        # many short prompts of odd lengths packed into one call
        dict(name="prompt_packed_40", kind="prompt", q_heads=32, kv_heads=8, head_dim=128, seqs=40, len_min=9, len_max=299,
             window=0, type="f16"),
        # the longest prompt, narrow heads
        dict(name="prompt_8192", kind="prompt", q_heads=32, kv_heads=8, head_dim=128, seqs=1, len_min=8192, len_max=8192,
             window=0, type="bf16"),
        # the distribution of one decoded token with its alternatives
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=262144, type="f32", cap=30.0, top=5),
        # a prompt piece scored over the whole vocabulary
        dict(name="logprobs_512", kind="logprobs", rows=512, vocab=262144, type="f32", cap=30.0, top=20),
        # a batch with an odd vocabulary and 16-bit logits, the given tokens only
        dict(name="logprobs_odd", kind="logprobs", rows=77, vocab=100003, type="bf16", cap=0.0, top=1),
        # between two blocks of one decoded token
        dict(name="norm_1", kind="norm", rows=1, hidden=2816, post=True, gate=False, out="f32"),
        # of a long prompt, the next projection's activations in bf16
        dict(name="norm_4096", kind="norm", rows=4096, hidden=2816, post=True, gate=True, out="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


HEADS = [(16, 8, 256), (32, 8, 128), (16, 16, 128), (8, 2, 256)]


def draw(rng):
    kind = rng.choice(["chunk", "prompt", "logprobs", "norm"])
    if kind == "chunk":
        qh, kvh, hd = rng.choice(HEADS)
        seqs = _log(rng, 1, 32)
        new_max = _log(rng, 1, 1024 if seqs <= 4 else 256)
        ctx_max = _log(rng, 16, 6000 if seqs <= 4 else 3000)
        return dict(kind=kind, q_heads=qh, kv_heads=kvh, head_dim=hd, seqs=seqs, new_min=rng.randint(1, new_max), new_max=new_max,
                    ctx_min=rng.randint(0, ctx_max), ctx_max=ctx_max, page=rng.choice([16, 16, 16, 8, 32, 64, 128, 256, 5, 24]),
                    window=rng.choice([0, 0, 0, rng.randint(1, 2000)]), q=rng.choice(["f32", "f16"]), out=rng.choice(["bf16", "f16"]))
    if kind == "prompt":
        qh, kvh, hd = rng.choice(HEADS)
        seqs = _log(rng, 1, 64)
        len_max = _log(rng, 8, 6000 // seqs + 8)
        return dict(kind=kind, q_heads=qh, kv_heads=kvh, head_dim=hd, seqs=seqs, len_min=rng.randint(1, len_max), len_max=len_max,
                    window=rng.choice([0, 0, 0, rng.randint(1, 2000)]), type=rng.choice(["bf16", "f16"]))
    if kind == "logprobs":
        return dict(kind=kind, rows=_log(rng, 1, 512), vocab=_log(rng, 1000, 262144), type=rng.choice(["f32", "f32", "f16", "bf16"]),
                    cap=rng.choice([0.0, 30.0, 50.0]), top=rng.choice([0, 1, 3, 5, 20, 64]))
    return dict(kind=kind, rows=_log(rng, 1, 8192), hidden=_log(rng, 256, 8192, rng.choice([1, 64, 256])), post=rng.random() < 0.6,
                gate=rng.random() < 0.5, out=rng.choice(["f32", "bf16"]))


# ---- what a program has in hand before the call ----
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + 17) & 0x7FFFFFFFFFFF)


def _spread(lo, hi, n, phase):
    """n whole numbers over [lo, hi], the same for every seed; the first is hi."""
    return [hi if i == 0 else lo + int((hi - lo + 1) * ((i * 0.6180339887 + phase) % 1.0)) for i in range(n)]


def _chunk_lengths(case):
    return _spread(case["new_min"], case["new_max"], case["seqs"], 0.1), _spread(case["ctx_min"], case["ctx_max"], case["seqs"], 0.7)


def _prompt_lengths(case):
    return _spread(case["len_min"], case["len_max"], case["seqs"], 0.3)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(lens):
    return [0] + [int(v) for v in np.cumsum(lens)]


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind == "chunk":
        new, ctx = _chunk_lengths(case)
        n, page, kvh, hd, qh = case["seqs"], case["page"], case["kv_heads"], case["head_dim"], case["q_heads"]
        need = [(a + b + page - 1) // page for a, b in zip(new, ctx)]
        blocks = sum(need) + 1
        # pages are handed out in the order sequences grew: a shuffle of the pool; block 0 is what unused entries point to
        order = (1 + torch.randperm(blocks - 1, generator=g, device=DEV)).to(torch.int32)
        s["table"] = torch.zeros((n, max(need)), dtype=torch.int32, device=DEV)
        at = 0
        for i, m in enumerate(need):
            s["table"][i, :m] = order[at:at + m]
            at += m
        # the new tokens' rows are in the cache already: the append comes before the attention
        s["k"] = torch.empty((blocks, page, kvh, hd), dtype=torch.float16, device=DEV).normal_(generator=g)
        s["v"] = torch.empty((blocks, page, kvh, hd), dtype=torch.float16, device=DEV).normal_(generator=g)
        s["start"], s["slot"], s["pos"] = _i32(_starts(new)), _i32(list(range(n))), _i32(ctx)
        rows = sum(new)
        # queries lie in front of each row of the fused projection output
        fused = torch.randn((rows, qh + 2 * kvh, hd), generator=g, device=DEV).to(TYPES[case["q"]])
        s["q"] = fused[:, :qh]
        s["out"] = torch.empty((rows, qh, hd), dtype=TYPES[case["out"]], device=DEV)
        s["scale"] = 1.0 / math.sqrt(hd)
        if own:  # the cache handle that such a program keeps, over the same pools and table
            from leviathan_b200 import PagedKV

            s["cache"] = PagedKV.over(s["k"], s["v"], s["table"])
    elif kind == "prompt":
        lens = _prompt_lengths(case)
        rows, kvh, hd, qh = sum(lens), case["kv_heads"], case["head_dim"], case["q_heads"]
        fused = torch.randn((rows, qh + 2 * kvh, hd), generator=g, device=DEV).to(TYPES[case["type"]])
        s["q"], s["k"], s["v"] = fused[:, :qh], fused[:, qh:qh + kvh], fused[:, qh + kvh:]
        s["start"] = _i32(_starts(lens))
        s["out"] = torch.empty((rows, qh, hd), dtype=TYPES[case["type"]], device=DEV)
        s["scale"] = 1.0 / math.sqrt(hd)
    elif kind == "logprobs":
        rows, n = case["rows"], case["vocab"]
        x = torch.randn((rows, n), generator=g, device=DEV) * 3.0
        s["tokens"] = torch.randint(0, n, (rows,), generator=g, device=DEV).to(torch.int32)
        # the given token is a likely one in most rows of real text
        x[torch.arange(rows, device=DEV), s["tokens"].long()] += 12.0 * torch.rand(rows, generator=g, device=DEV)
        s["logits"] = x.to(TYPES[case["type"]])
    else:
        rows, n = case["rows"], case["hidden"]
        s["x"] = torch.randn((rows, n), generator=g, device=DEV) * 0.7
        s["residual"] = torch.randn((rows, n), generator=g, device=DEV) * 2.0
        s["post"] = 1.0 + 0.1 * torch.randn(n, generator=g, device=DEV) if case["post"] else None
        s["pre"] = 1.0 + 0.1 * torch.randn(n, generator=g, device=DEV)
        s["gate"] = torch.rand(n, generator=g, device=DEV) if case["gate"] else None
        s["alpha"], s["scale"], s["eps"] = 0.9, 1.1, 1e-6
        s["res_out"] = torch.empty_like(s["residual"])
        s["h"] = torch.empty((rows, n), dtype=TYPES[case["out"]], device=DEV)
    return s


# ---- plain forms ----
def _softmax_values(q, k, v, allowed, scale):
    """q [.., g * m, d], k, v [.., n, d], allowed broadcast over [.., g * m, n]."""
    w = torch.matmul(q, k.transpose(-1, -2)) * scale
    w = w.masked_fill_(~allowed, -math.inf)
    w = torch.exp(w.sub_(w.amax(-1, keepdim=True)))
    return torch.matmul(w, v) / w.sum(-1, keepdim=True)


def _plain_chunk(s):
    q, start, pos = s["q"].float(), s["start"].long(), s["pos"].long()
    rows, qh, hd = q.shape
    n, kvh, page, window = start.numel() - 1, s["k"].shape[2], s["k"].shape[1], s["case"]["window"]
    g = qh // kvh
    row = torch.arange(rows, device=DEV)
    seq = torch.bucketize(row, start[1:], right=True)
    off = row - start[seq]
    most = s["case"]["new_max"]
    entries = s["table"][s["slot"].long()].long()
    k = s["k"][entries].float().view(n, -1, kvh, hd).permute(0, 2, 1, 3)
    v = s["v"][entries].float().view(n, -1, kvh, hd).permute(0, 2, 1, 3)
    qp = torch.zeros((n, most, qh, hd), device=DEV)
    qp[seq, off] = q
    qp = qp.view(n, most, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * most, hd)
    at = (pos[:, None] + torch.arange(most, device=DEV))[:, None, :, None]
    j = torch.arange(k.shape[2], device=DEV)
    allowed = j <= at
    if window:
        allowed &= j > at - window
    o = _softmax_values(qp, k, v, allowed.repeat(1, 1, g, 1), s["scale"])
    o = o.view(n, kvh, g, most, hd).permute(0, 3, 1, 2, 4).reshape(n, most, qh, hd)
    return o[seq, off].to(TYPES[s["case"]["out"]])


def _plain_prompt(s):
    rows, qh, hd = s["q"].shape
    kvh = s["k"].shape[1]
    g = qh // kvh
    q = s["q"].float().view(rows, kvh, g, hd).permute(1, 2, 0, 3).reshape(kvh, g * rows, hd)
    k, v = s["k"].float().permute(1, 0, 2), s["v"].float().permute(1, 0, 2)
    row = torch.arange(rows, device=DEV)
    seq = torch.bucketize(row, s["start"].long()[1:], right=True)
    allowed = (seq[:, None] == seq[None, :]) & (row[None, :] <= row[:, None])
    if s["case"]["window"]:
        allowed &= row[None, :] > row[:, None] - s["case"]["window"]
    o = _softmax_values(q, k, v, allowed.repeat(g, 1)[None], s["scale"])
    return o.view(kvh, g, rows, hd).permute(2, 0, 1, 3).reshape(rows, qh, hd).to(s["q"].dtype)


def _order_key(raw):
    """Whole numbers in the order of the values, larger ones for lower indices where values tie."""
    b = raw.contiguous().view(torch.int32).to(torch.int64)
    b = torch.where(b < 0, -(b & 0x7FFFFFFF), b)  # sign and magnitude to a whole number: -0 and 0 are the same
    return b * (1 << 24) - torch.arange(raw.shape[1], device=raw.device)


def _plain_logprobs(s):
    raw, top, cap = s["logits"].float(), s["case"]["top"], s["case"]["cap"]
    x = cap * torch.tanh(raw / cap) if cap else raw
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    out = {"logprob": (x.gather(1, s["tokens"].long()[:, None]) - lse)[:, 0], "entropy": (lse - (e * x).sum(-1, keepdim=True) / z)[:, 0]}
    if top:
        ids = torch.topk(_order_key(raw), top, dim=1).indices
        out["top_index"] = ids.to(torch.int32)
        out["top_logprob"] = x.gather(1, ids) - lse
    return out


def _plain_norm(s):
    b = s["x"]
    if s["post"] is not None:
        b = b / torch.sqrt((b * b).mean(-1, keepdim=True) + s["eps"]) * s["post"]
    if s["gate"] is not None:
        b = b * s["gate"]
    r = s["scale"] * (s["residual"] + s["alpha"] * b)
    h = r / torch.sqrt((r * r).mean(-1, keepdim=True) + s["eps"]) * s["pre"]
    return r, h.to(TYPES[s["case"]["out"]])


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import leviathan_b200

        _ctx = leviathan_b200.Context(0)
    return _ctx


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"chunk": _plain_chunk, "prompt": _plain_prompt, "logprobs": _plain_logprobs, "norm": _plain_norm}[kind](s)
    ctx = _context()
    if kind == "chunk":
        return ctx.attn_chunk(s["cache"], s["start"], s["slot"], s["pos"], s["q"], case["window"], s["scale"], out=s["out"])
    if kind == "prompt":
        return ctx.attn_prompt(s["q"], s["k"], s["v"], s["start"], case["window"], s["scale"], out=s["out"])
    if kind == "logprobs":
        lp, ent, ids, tops = ctx.logprobs(s["logits"], s["tokens"], top=case["top"], softcap=case["cap"])
        return dict(logprob=lp, entropy=ent, **(dict(top_index=ids, top_logprob=tops) if case["top"] else {}))
    return ctx.norm_residual(s["x"], s["residual"], post=s["post"], pre=s["pre"], gate=s["gate"], alpha=s["alpha"], scale=s["scale"],
                             eps=s["eps"], out=s["res_out"], h=s["h"])


# ---- what a pass cannot do without ----
def _attended(ctx, new, window):
    """Positions that the rows of one sequence attend to, summed, and how many distinct ones there are."""
    p = np.arange(ctx, ctx + new, dtype=np.int64)
    lo = np.maximum(0, p + 1 - window) if window else np.zeros_like(p)
    return int((p + 1 - lo).sum()), int(ctx + new - lo[0])


def work(case):
    kind = case["kind"]
    if kind in ("chunk", "prompt"):
        new, ctx = _chunk_lengths(case) if kind == "chunk" else (_prompt_lengths(case), [0] * case["seqs"])
        total, distinct = (sum(v) for v in zip(*(_attended(c, n, case["window"]) for n, c in zip(new, ctx))))
        qn, size = sum(new) * case["q_heads"] * case["head_dim"], 4 if case.get("q") == "f32" else 2
        return dict(bytes=qn * (size + 2) + 4 * distinct * case["kv_heads"] * case["head_dim"], flops=4.0 * total * case["q_heads"] * case["head_dim"])
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (4 if case["type"] == "f32" else 2) + case["rows"] * (12 + 8 * case["top"]), flops=(8.0 if case["cap"] else 4.0) * n)
    n = case["rows"] * case["hidden"]
    return dict(bytes=n * (12 + (4 if case["out"] == "f32" else 2)) + 4 * case["hidden"] * (1 + case["post"] + case["gate"]), flops=10.0 * n)


# ---- the definition in 64 bits ----
def _exact_attention(q, k, v, first, window, scale):
    """One sequence: q [m][heads][d] at positions first, first + 1, ...; k, v [n][kv heads][d] from position 0 on."""
    m, qh, _ = q.shape
    g = qh // k.shape[1]
    out = torch.empty((m, qh, q.shape[2]), dtype=torch.float64, device=DEV)
    p = first + torch.arange(m, device=DEV)[:, None]
    j = torch.arange(k.shape[0], device=DEV)[None, :]
    hidden = (j > p) | (j <= p - window) if window else j > p
    for h in range(qh):
        logits = (q[:, h].double() @ k[:, h // g].double().T) * scale
        logits[hidden] = -math.inf
        out[:, h] = torch.softmax(logits, -1) @ v[:, h // g].double()
    return out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "chunk":
        new, ctx = _chunk_lengths(case)
        at, parts, page = 0, [], case["page"]
        for i, (m, c) in enumerate(zip(new, ctx)):
            total = m + c
            e = s["table"][i, :(total + page - 1) // page].long()
            rows = [s[w].index_select(0, e).flatten(0, 1)[:total] for w in ("k", "v")]
            parts.append(_exact_attention(s["q"][at:at + m], rows[0], rows[1], c, case["window"], s["scale"]))
            at += m
        return torch.cat(parts)
    if kind == "prompt":
        at, parts = 0, []
        for m in _prompt_lengths(case):
            part = slice(at, at + m)
            parts.append(_exact_attention(s["q"][part], s["k"][part], s["v"][part], 0, case["window"], s["scale"]))
            at += m
        return torch.cat(parts)
    if kind == "logprobs":
        got = {"logprob": [], "entropy": [], "top_index": [], "top_logprob": []}
        for r in range(case["rows"]):
            raw = s["logits"][r].double()
            x = case["cap"] * torch.tanh(raw / case["cap"]) if case["cap"] else raw
            lp = torch.log_softmax(x, 0)
            got["logprob"].append(lp[s["tokens"][r].long()])
            got["entropy"].append(torch.where(lp > -math.inf, -torch.exp(lp) * lp, 0.0).sum())
            ids = torch.sort(raw, descending=True, stable=True).indices[:case["top"]]
            got["top_index"].append(ids.to(torch.int32))
            got["top_logprob"].append(lp[ids])
        return {k: torch.stack(v) for k, v in got.items() if case["top"] or not k.startswith("top")}
    x, res = s["x"].double(), s["residual"].double()
    if s["post"] is not None:
        x = x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + s["eps"]) * s["post"].double()
    if s["gate"] is not None:
        x = x * s["gate"].double()
    r = (res + x * s["alpha"]) * s["scale"]
    return r, r * torch.rsqrt(r.pow(2).mean(1, keepdim=True) + s["eps"]) * s["pre"].double()
