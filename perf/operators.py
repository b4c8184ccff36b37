"""Measured cases of the speculative decode step's operators.

The step, as a serving program runs it for every stream of a talker (or code
predictor) without returning to the host: map pages of the 4-bit KV cache for
the new tokens (`tables`), norm and rotate q and k and append k and v in 4 bits
(`append`), attend over the 4-bit cache (`attend`), turn logits into the
sampler's probabilities (`probs`), and verify the drafted tokens against them
(`verify`).

`run` computes an operator in its plain form (elementary torch operations) or,
where `own` is true, through the calls a user makes of qora_b200.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6      # of the per-head RMS norm
THETA = 1e6     # RoPE base
ROPE_MAX = 32768


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # block tables and slot maps: a decode step of 32 streams with caches of up to 4096 positions
        dict(name="tables_32", kind="tables", streams=32, max_pos=4608, page=64, ctx=4096, count=1, prompts=0),
        # a large serving batch: 512 streams of up to 32768 positions, drafts of 0..5 tokens, and
        # three admitted prompts
        dict(name="tables_512", kind="tables", streams=512, max_pos=32768, page=32, ctx=32768, count=5, prompts=3),
        # append of one token for each of 32 streams (a decode step at batch 32)
        dict(name="append_32", kind="append", tokens=32, heads=16, kv_heads=8, head_dim=128, page=64, pad=0),
        # append of prompts: 8191 tokens, rows behind them padded
        dict(name="append_8191", kind="append", tokens=8191, heads=16, kv_heads=8, head_dim=128, page=64, pad=33),
        # one stream's decode step, the latency case
        dict(name="attend_1x700", kind="attend", streams=1, heads=16, kv_heads=8, head_dim=128, page=64,
             ctx=700, ragged=False, mode="one", count=1),
        # a decode step of 32 streams with 4096 positions each
        dict(name="attend_32x4096", kind="attend", streams=32, heads=16, kv_heads=8, head_dim=128, page=64,
             ctx=4096, ragged=False, mode="one", count=1),
        # ragged streams of up to 12288 positions that verify 0..5 drafted tokens
        dict(name="attend_drafts", kind="attend", streams=40, heads=16, kv_heads=8, head_dim=128, page=128,
             ctx=12288, ragged=True, mode="draft", count=6),
        # two prompts on top of short caches
        dict(name="attend_prompt", kind="attend", streams=2, heads=16, kv_heads=8, head_dim=128, page=64,
             ctx=300, ragged=True, mode="prompt", count=2048),
        # the sampler's probabilities over the predictor's vocabulary, 32 streams x 5 positions
        dict(name="probs_160x2048", kind="probs", rows=160, vocab=2048, top_k=50, top_p=1.0, temperature=0.9, penalty=1.05, prev=16),
        # over a text vocabulary
        dict(name="probs_96x151936", kind="probs", rows=96, vocab=151936, top_k=50, top_p=0.95, temperature=0.8, penalty=1.1, prev=64),
        # verification of 4 drafts for 32 streams over the predictor's vocabulary
        dict(name="verify_32x4x2048", kind="verify", streams=32, drafts=4, vocab=2048, dist=True, agree=0.7),
        # of 5 drafts for 64 streams over a text vocabulary
        dict(name="verify_64x5x151936", kind="verify", streams=64, drafts=5, vocab=151936, dist=True, agree=0.8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attend", "attend", "probs", "verify"])
    if kind == "tables":
        page = rng.choice([32, 64, 128])
        return dict(kind=kind, streams=_log(rng, 1, 512), max_pos=32768, page=page, ctx=_log(rng, 64, 32000),
                    count=rng.randint(1, 9), prompts=rng.randint(0, 3))
    heads, kv_heads = rng.choice([(16, 8), (4, 2), (16, 16), (8, 2), (32, 8), (6, 2)])
    head_dim = rng.choice([64, 128])
    page = rng.choice([32, 64, 128])
    if kind == "append":
        tokens = _log(rng, 1, 6000)
        return dict(kind=kind, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    pad=rng.choice([0, 7]))
    if kind == "attend":
        mode = rng.choice(["one", "one", "draft", "draft", "prompt"])
        if mode == "prompt":
            streams, ctx, count = rng.randint(1, 3), rng.randint(0, 500), _log(rng, 17, 1100)
        else:
            ctx = _log(rng, 1, 12000)
            streams = max(1, min(_log(rng, 1, 64), 130000 // ctx))
            count = 1 if mode == "one" else rng.randint(2, 9)
        return dict(kind=kind, streams=streams, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    ctx=ctx, ragged=rng.random() < 0.7, mode=mode, count=count)
    vocab = rng.choice([_log(rng, 65, 8192), _log(rng, 8192, 151936)])
    if kind == "probs":
        rows = max(1, min(_log(rng, 1, 512), 14000000 // vocab))
        top_k = rng.choice([0, 1, 40, 50, 50, 200, 1000])
        return dict(kind=kind, rows=rows, vocab=vocab, top_k=top_k,
                    top_p=rng.choice([1.0, 0.9, 0.95]) if 0 < top_k < vocab else 1.0,
                    temperature=rng.choice([0.7, 0.9, 1.0, 1.3]), penalty=rng.choice([1.0, 1.05, 1.2]),
                    prev=rng.choice([0, 16, 33]))
    drafts = rng.randint(1, 8)
    return dict(kind=kind, streams=max(1, min(_log(rng, 1, 128), 50000000 // (vocab * (drafts + 1)))),
                drafts=drafts, vocab=vocab, dist=rng.random() < 0.75, agree=rng.choice([0.3, 0.8, 0.97]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)


def _package():
    pkg = os.path.join(os.getcwd(), "qora-tts-12hz-1.7b_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from qora_b200 import engine, kv4
    return engine, kv4


_ctx = None


def _context(engine):
    global _ctx
    if _ctx is None:
        _ctx = engine.Context(torch.cuda.current_device())
    return _ctx


def _table(g, lens, page, per_stream, pool):
    """A fragmented block table: the streams' pages are scattered over the pool; -1 where none is mapped."""
    keep = (lens + page - 1) // page
    at = torch.cumsum(keep, 0) - keep
    order = torch.randperm(pool, generator=g, device=DEV)
    j = torch.arange(per_stream, device=DEV)
    take = (at[:, None] + j).clamp(max=pool - 1)
    return torch.where(j < keep[:, None], order[take], -1).to(torch.int32)


def _rope(head_dim):
    half = head_dim // 2
    freq = THETA ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / head_dim)
    ang = torch.arange(ROPE_MAX, device=DEV, dtype=torch.float64)[:, None] * freq
    return torch.cos(ang).float().contiguous(), torch.sin(ang).float().contiguous()


def _quantise(x):
    """Groups of 32: scale f16(amax / 7), codes the nearest integers to x / scale."""
    grp = x.double().unflatten(-1, (-1, 32))
    scale = (grp.abs().amax(-1) / 7).float().half().clamp(max=65504.0)
    s = scale.double()[..., None]
    codes = torch.where(s > 0, torch.round(grp / torch.where(s > 0, s, 1.0)), 0.0).clamp(-7, 7)
    return codes.to(torch.int8).flatten(-2), scale


def _counts(case, g):
    """New tokens of each stream: the case gives how many there are of each count, the seed who has them."""
    S, n, fixed = case["streams"], case["count"], _gen(7)
    if case["kind"] == "tables":
        c = _ints(fixed, 0 if n > 1 else 1, n + 1, (S,))
        for p in range(min(case["prompts"], S)):
            c[p * (S // 3) % S] = 200 + 331 * p
    elif case["mode"] == "one":
        return torch.ones(S, dtype=torch.int32, device=DEV)
    elif case["mode"] == "draft":
        c = _ints(fixed, 0, n + 1, (S,))
        c[S // 2] = n
    else:
        c = _ints(fixed, max(1, n // 2), n + 1, (S,))
        c[0] = n
    return c[torch.randperm(S, generator=g, device=DEV)].contiguous()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = dict(case=dict(case))
    if kind == "tables":
        S, P, per = case["streams"], case["page"], -(-case["max_pos"] // case["page"])
        lens = _ints(g, 0, case["ctx"] + 1, (S,)).clamp(max=case["max_pos"] - 1000)
        counts = _counts(case, g)
        tokens = int(counts.sum()) + 5
        pages = int(((lens + P - 1) // P).sum())
        pool = pages + pages // 8 + int(((counts + P - 1) // P + 1).sum())
        st.update(lens=lens, counts=counts, pool=pool, max_tokens=tokens, table=_table(g, lens, P, per, pool))
        if own:
            engine, kv4 = _package()
            kv = kv4.Kv4Cache(_context(engine), 1, 1, 1, 64, case["max_pos"], S, P, pool)
            s = kv.state()
            s["table"].copy_(st["table"])
            s["lengths"].copy_(lens)
            st.update(kv=kv, kv_table=s["table"], slots=torch.empty(tokens, dtype=torch.int32, device=DEV),
                      positions=torch.empty(tokens, dtype=torch.int32, device=DEV),
                      offsets=torch.empty(S + 1, dtype=torch.int32, device=DEV))
    elif kind == "append":
        H, KV, D, P, N = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["tokens"]
        pool = -(-N // P) + 3
        qkv = torch.randn(N + case["pad"], (H + 2 * KV) * D, generator=g, device=DEV)
        qkv = qkv * torch.exp(0.5 * torch.randn(N + case["pad"], 1, generator=g, device=DEV))
        slots = torch.randperm(pool * P, generator=g, device=DEV)[:N + case["pad"]].to(torch.int32).contiguous()
        if case["pad"]:
            slots[N:] = -1
        cos, sin = _rope(D)
        st.update(qkv=qkv, slots=slots, positions=_ints(g, 0, ROPE_MAX, (N + case["pad"],)), cos=cos, sin=sin,
                  q_norm=(1 + 0.1 * torch.randn(D, generator=g, device=DEV)).half(),
                  k_norm=(1 + 0.1 * torch.randn(D, generator=g, device=DEV)).half())
        if own:
            engine, kv4 = _package()
            rows = N + case["pad"]
            st.update(kv=kv4.Kv4Cache(_context(engine), 1, H, KV, D, pool * P, 1, P, pool),
                      q=torch.zeros(rows, H * D, device=DEV), k=torch.zeros(rows, KV * D, device=DEV),
                      v=torch.zeros(rows, KV * D, device=DEV))
    elif kind == "attend":
        H, KV, D, P, S = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["streams"]
        lens = _ints(g, 0, case["ctx"] + 1, (S,)) if case["ragged"] else torch.full((S,), case["ctx"], dtype=torch.int32, device=DEV)
        if case["ragged"]:
            lens[0] = case["ctx"]
        counts = _counts(case, g)
        total = lens + counts
        N, longest = int(counts.sum()), int(total.max())
        per = -(-longest // P)
        pool = int(((total + P - 1) // P).sum()) + 3
        kc = torch.empty(pool * P, KV, D, dtype=torch.int8, device=DEV)
        vc = torch.empty_like(kc)
        ks = torch.empty(pool * P, KV, D // 32, dtype=torch.float16, device=DEV)
        vs = torch.empty_like(ks)
        for at in range(0, pool * P, 65536):
            rows = slice(at, min(at + 65536, pool * P))
            n = rows.stop - at
            kc[rows], ks[rows] = _quantise(torch.randn(n, KV, D, generator=g, device=DEV))
            vc[rows], vs[rows] = _quantise(torch.randn(n, KV, D, generator=g, device=DEV) + 0.1)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), torch.cumsum(counts, 0).to(torch.int32)])
        st.update(q=1.5 * torch.randn(N, H * D, generator=g, device=DEV), lens=lens, counts=counts, offsets=offsets, longest=longest,
                  most=int(counts.max()), k_codes=kc, k_scales=ks, v_codes=vc, v_scales=vs,
                  table=_table(g, total, P, per, pool))
        if own:
            engine, kv4 = _package()
            kv = kv4.Kv4Cache(_context(engine), 1, H, KV, D, per * P, S, P, pool)
            s = kv.state()
            s["table"].copy_(st["table"])
            s["lengths"].copy_(lens)
            slot = torch.arange(pool * P, dtype=torch.int32, device=DEV)
            for at in range(0, pool * P, 65536):
                rows = slice(at, min(at + 65536, pool * P))
                kv.write(0, slot[rows], (kc[rows].unflatten(-1, (-1, 32)) * ks[rows].float()[..., None]).flatten(1),
                         (vc[rows].unflatten(-1, (-1, 32)) * vs[rows].float()[..., None]).flatten(1))
            st.update(kv=kv, out=torch.empty(N, H * D, device=DEV))
    elif kind == "probs":
        R, V = case["rows"], case["vocab"]
        logits = 3.0 * torch.randn(R, V, generator=g, device=DEV)
        logits[:, V // 3:V // 3 + max(1, V // 50)] = -math.inf      # tokens that a program forbids
        prev = _ints(g, 0, V, (R, case["prev"])) if case["prev"] else None
        if prev is not None and case["prev"] > 3:
            prev[:, 1] = prev[:, 0]                                    # a token said twice
            prev[:, 2] = logits.argmax(-1).to(torch.int32)
        st.update(logits=logits, prev=prev)
        if own:
            engine, _ = _package()
            st.update(engine=engine, ctx=_context(engine), out=torch.empty(R, V, device=DEV),
                      params=engine._lib.SampleParams(case["temperature"], case["top_k"], case["top_p"], case["penalty"]))
    else:
        S, K, V = case["streams"], case["drafts"], case["vocab"]
        target = 2.5 * torch.randn(S, K + 1, V, generator=g, device=DEV)
        near = case["agree"] * target[:, :K] + (1 - case["agree"] ** 2) ** 0.5 * 2.5 * torch.randn(S, K, V, generator=g, device=DEV)
        noise = torch.rand(S, K, V, generator=g, device=DEV).clamp_(1e-30)
        drafts = (near - torch.log(-torch.log(noise).clamp_(1e-30))).argmax(-1).to(torch.int32)   # drawn from the draft's distribution
        counts = _ints(g, 0, K + 1, (S,))
        counts[: (S + 1) // 2] = K
        st.update(drafts=drafts.contiguous(), target=torch.softmax(target, -1), draft=torch.softmax(near, -1) if case["dist"] else None,
                  counts=counts, uniforms=torch.rand(S, K + 1, generator=g, device=DEV))
        if own:
            engine, _ = _package()
            st.update(engine=engine, ctx=_context(engine), tokens=torch.empty(S, K + 1, dtype=torch.int32, device=DEV),
                      n_out=torch.empty(S, dtype=torch.int32, device=DEV))
    return st


# ------------------------------------------------------------------ the plain forms
def _tables(st):
    c, lens, counts, table = st["case"], st["lens"].long(), st["counts"].long(), st["table"].long()
    P, S, pool = c["page"], c["streams"], st["pool"]
    keep, want = (lens + P - 1) // P, (lens + counts + P - 1) // P
    j = torch.arange(table.shape[1], device=DEV)
    used = torch.zeros(pool + 1, dtype=torch.bool, device=DEV)
    used[torch.where(j < keep[:, None], table, pool)] = True
    free = ~used[:pool]
    rank = torch.cumsum(free.long(), 0) - 1
    listing = torch.zeros(pool + 1, dtype=torch.long, device=DEV)
    listing[torch.where(free, rank, pool)] = torch.arange(pool, device=DEV)
    need = want - keep
    at = torch.cumsum(need, 0) - need
    new = (j >= keep[:, None]) & (j < want[:, None])
    table = torch.where(new, listing[(at[:, None] + j - keep[:, None]).clamp(0, pool)], table)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(counts, 0)])
    i = torch.arange(st["max_tokens"], device=DEV)
    b = (torch.searchsorted(offsets, i, right=True) - 1).clamp(max=S - 1)
    inside = i < offsets[-1]
    pos = torch.where(inside, lens[b] + i - offsets[b], 0)
    slots = torch.where(inside, table[b, pos // P] * P + pos % P, -1)
    return dict(table=table.int(), slots=slots.int(), positions=pos.int(), offsets=offsets.int())


def _normed(x, gamma, cos, sin):
    """Per-head RMS norm and split rotation, in 64 bits (4-bit codes sit next to borders)."""
    x = x.double()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.double()
    a, b = x.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1).float()


def _append(st):
    c = st["case"]
    H, KV, D = c["heads"], c["kv_heads"], c["head_dim"]
    N = st["qkv"].shape[0]
    live = (st["slots"] >= 0)[:, None]
    q, k, v = st["qkv"].split([H * D, KV * D, KV * D], -1)
    at = st["positions"].long()
    cos, sin = st["cos"][at], st["sin"][at]
    q = _normed(q.view(N, H, D), st["q_norm"], cos, sin)
    held = []
    for x in (_normed(k.view(N, KV, D), st["k_norm"], cos, sin), v.view(N, KV, D)):
        codes, scale = _quantise(x)
        held.append((codes.unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(1))
    return dict(q=torch.where(live, q.flatten(1), 0.0), k=torch.where(live, held[0], 0.0), v=torch.where(live, held[1], 0.0))


def _attend(st):
    c = st["case"]
    H, KV, D, P, S = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["streams"]
    L, T, G = st["longest"], st["most"], c["heads"] // c["kv_heads"]
    lens, counts, offsets = st["lens"].long(), st["counts"].long(), st["offsets"].long()
    pos = torch.arange(L, device=DEV)
    slot = st["table"].long()[:, pos // P].clamp(min=0) * P + pos % P                         # [S][L]
    k = (st["k_codes"][slot].unflatten(-1, (-1, 32)) * st["k_scales"][slot].float()[..., None]).flatten(-2)
    t = torch.arange(T, device=DEV)
    row = (offsets[:-1, None] + t).clamp(max=st["q"].shape[0] - 1)                            # [S][T]
    q = st["q"][row].view(S, T, KV, G, D).permute(0, 2, 3, 1, 4).reshape(S, KV, G * T, D)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).view(S, KV, G, T, L) * (D ** -0.5)
    del k
    seen = pos <= (lens[:, None] + t)[..., None]                                              # [S][T][L]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    del s
    p = (p / p.sum(-1, keepdim=True)).view(S, KV, G * T, L)
    v = (st["v_codes"][slot].unflatten(-1, (-1, 32)) * st["v_scales"][slot].float()[..., None]).flatten(-2)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)).view(S, KV, G, T, D).permute(0, 3, 1, 2, 4).reshape(S * T, H * D)
    out = torch.zeros(st["q"].shape[0] + 1, H * D, device=DEV)
    out[torch.where(t < counts[:, None], row, st["q"].shape[0]).view(-1)] = o
    return dict(out=out[:-1])


def _probs(st):
    c = st["case"]
    x, V = st["logits"].double(), c["vocab"]
    if st["prev"] is not None and c["penalty"] != 1.0:
        said = torch.zeros_like(x).scatter_add_(1, st["prev"].long(), torch.ones_like(st["prev"], dtype=torch.float64))
        times = torch.full_like(x, _f32(c["penalty"])) ** said
        x = torch.where(x > 0, x / times, torch.where(said > 0, x * times, x))
    z = x / _f32(c["temperature"])
    if 0 < c["top_k"] < V:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : c["top_k"]]
        z = z.gather(1, order)
    e = torch.exp(z - z.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    if 0 < c["top_k"] < V:
        if 0 < c["top_p"] < 1:
            before = torch.cumsum(p, -1) - p
            p = torch.where(before < _f32(c["top_p"]), p, 0.0)
            p = p / p.sum(-1, keepdim=True)
        p = torch.zeros_like(x).scatter_(1, order, p)
    return dict(probs=p.float())


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _verify(st):
    c = st["case"]
    S, K, V = c["streams"], c["drafts"], c["vocab"]
    drafts, target, draft, u, counts = st["drafts"].long(), st["target"], st["draft"], st["uniforms"].double(), st["counts"].long()
    p = target[:, :K].gather(-1, drafts[..., None])[..., 0].double()
    q = draft.gather(-1, drafts[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    i = torch.arange(K, device=DEV)
    passed = (u[:, :K] * q < p) & (i < counts[:, None])
    a = torch.cumprod(passed.long(), -1).sum(-1)
    rows = torch.arange(S, device=DEV)
    w = target[rows, a].double()
    rejected = (a < counts)[:, None]
    at = a.clamp(max=K - 1)
    if draft is not None:
        rest = (w - draft[rows, at].double()).clamp(min=0)
    else:
        rest = w.scatter(1, drafts[rows, at][:, None], 0.0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    w = torch.where(rejected, rest, w)
    cum = torch.cumsum(w, -1)
    over = cum > (u[:, K] * cum[:, -1])[:, None]
    index = torch.arange(V, device=DEV)
    last = torch.where(w > 0, index, 0).amax(-1)
    token = torch.where(over.any(-1), torch.where(over, index, V).amin(-1), last)
    j = torch.arange(K + 1, device=DEV)
    said = torch.where(j < a[:, None], torch.cat([drafts, drafts[:, :1]], 1), -1)
    said = torch.where(j == a[:, None], token[:, None], said)
    return dict(tokens=said.int(), n_out=(a + 1).int())


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"tables": _tables, "append": _append, "attend": _attend, "probs": _probs, "verify": _verify}[kind](st)
    if kind == "tables":
        st["kv"].reserve(st["counts"], st["max_tokens"], out=(st["slots"], st["positions"], st["offsets"]))
        return dict(table=st["kv_table"], slots=st["slots"], positions=st["positions"], offsets=st["offsets"])
    if kind == "append":
        st["kv"].append(0, st["qkv"], st["q_norm"], st["k_norm"], st["cos"], st["sin"], st["positions"], st["slots"], out=st["q"])
        st["kv"].read(0, st["slots"], out=(st["k"], st["v"]))
        return dict(q=st["q"], k=st["k"], v=st["v"])
    if kind == "attend":
        st["kv"].attend(0, st["q"], st["offsets"], st["most"], out=st["out"])
        return dict(out=st["out"])
    if kind == "probs":
        st["engine"].sample_probs(st["ctx"], st["logits"], st["prev"], st["params"], out=st["out"])
        return dict(probs=st["out"])
    st["engine"].verify_drafts(st["ctx"], st["drafts"], st["draft"], st["target"], st["uniforms"], st["counts"],
                               out=(st["tokens"], st["n_out"]))
    return dict(tokens=st["tokens"], n_out=st["n_out"])


# ------------------------------------------------------------------ floors
def _expected_lengths(case):
    """Positions that the streams hold together, and tokens, as the case draws them on average."""
    S = case["streams"]
    ctx = case["ctx"] if case.get("ragged") is False else case["ctx"] / 2
    n = {"one": 1.0, "draft": case["count"] / 2, "prompt": 0.75 * case["count"]}[case["mode"]]
    return S, ctx, n


def work(case):
    kind = case["kind"]
    if kind == "tables":
        S = case["streams"]
        tokens = S * (case["count"] + 1) / 2 + 500 * case["prompts"]
        return dict(bytes=4 * (3 * S + S * case["ctx"] / 2 / case["page"] + 2 * tokens), flops=0)
    if kind == "append":
        H, KV, D, N = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
        row = 4 * (H + 2 * KV) * D + 4 * H * D + 2 * KV * (D // 2 + D // 16)
        return dict(bytes=N * row, flops=N * (8 * (H + KV) * D + 4 * KV * D))
    if kind == "attend":
        H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
        S, ctx, n = _expected_lengths(case)
        return dict(bytes=S * ((ctx + n) * KV * 2 * (D // 2 + D // 16) + n * 8 * H * D),
                    flops=4 * H * D * S * n * (ctx + (n + 1) / 2))
    if kind == "probs":
        return dict(bytes=8 * case["rows"] * case["vocab"], flops=4 * case["rows"] * case["vocab"])
    return dict(bytes=4 * case["streams"] * (case["vocab"] * (1.5 if case["dist"] else 1) + 4 * case["drafts"]),
                flops=3 * case["streams"] * case["vocab"])


# ------------------------------------------------------------------ the definition in 64 bits
def _held(x):
    """What groups of 32 of the float32 rows x [..][D] stand for in 4 bits: code times scale."""
    x = x.to(torch.float64)
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], 32):
        part = x[..., at:at + 32]
        step = (part.abs().max(-1, keepdim=True)[0] / 7.0).to(torch.float32).to(torch.float16).to(torch.float64)
        out[..., at:at + 32] = torch.where(step == 0, torch.zeros_like(part), step * torch.round(part / step).clamp(-7, 7))
    return out


def _exact_append(st, case):
    H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
    rows = st["qkv"].to(torch.float64)
    cos, sin = st["cos"].to(torch.float64)[st["positions"].long()], st["sin"].to(torch.float64)[st["positions"].long()]
    dead = st["slots"] < 0

    def turned(head, gamma):
        x = rows[:, head * D:(head + 1) * D]
        x = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / D + EPS) * gamma.to(torch.float64)
        first, second = x[:, :D // 2], x[:, D // 2:]
        return torch.hstack([first * cos - second * sin, first * sin + second * cos])

    q = torch.hstack([turned(h, st["q_norm"]) for h in range(H)])
    k = torch.hstack([_held(turned(H + h, st["k_norm"]).to(torch.float32)) for h in range(KV)])
    v = torch.hstack([_held(rows[:, (H + KV + h) * D:(H + KV + h + 1) * D]) for h in range(KV)])
    for x in (q, k, v):
        x[dead] = 0
    return dict(q=q, k=k, v=v)


def _exact_attend(st, case):
    H, KV, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(st["q"].shape[0], H, D, dtype=torch.float64, device=DEV)
    lens, counts, offsets = st["lens"].tolist(), st["counts"].tolist(), st["offsets"].tolist()
    for b, (held, new) in enumerate(zip(lens, counts)):
        if not new:
            continue
        all_pages = st["table"][b, :-(-(held + new) // P)].long()
        where = (all_pages[:, None] * P + torch.arange(P, device=DEV)).flatten()[:held + new]
        q = st["q"][offsets[b]:offsets[b] + new].view(new, H, D).to(torch.float64)
        hidden = torch.arange(held + new, device=DEV)[None] > held + torch.arange(new, device=DEV)[:, None]
        for h in range(KV):
            k = st["k_codes"][where, h].to(torch.float64) * st["k_scales"][where, h].to(torch.float64).repeat_interleave(32, -1)
            v = st["v_codes"][where, h].to(torch.float64) * st["v_scales"][where, h].to(torch.float64).repeat_interleave(32, -1)
            for g in range(h * (H // KV), (h + 1) * (H // KV)):
                score = (q[:, g] @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[offsets[b]:offsets[b] + new, g] = torch.softmax(score, -1) @ v
    return dict(out=out.flatten(1))


def _exact_probs(st, case):
    x = st["logits"].to(torch.float64).clone()
    penalty, temperature, top_p = (float(torch.tensor(case[n], dtype=torch.float32)) for n in ("penalty", "temperature", "top_p"))
    if st["prev"] is not None and case["penalty"] != 1.0:
        every = torch.arange(x.shape[0], device=DEV)
        for n in range(case["prev"]):
            at = st["prev"][:, n].long()
            was = x[every, at]
            x[every, at] = torch.where(was > 0, was / penalty, was * penalty)
    p = torch.softmax(x / temperature, -1)
    if 0 < case["top_k"] < case["vocab"]:
        # among equal logits the lower index comes first
        order = torch.argsort(-x, dim=-1, stable=True)
        sorted_p = p.gather(1, order)
        sorted_p[:, case["top_k"]:] = 0
        sorted_p = sorted_p / sorted_p.sum(-1, keepdim=True)
        if 0 < case["top_p"] < 1:
            sorted_p[:, 1:][torch.cumsum(sorted_p, -1)[:, :-1] >= top_p] = 0
            sorted_p = sorted_p / sorted_p.sum(-1, keepdim=True)
        p = torch.zeros_like(p).scatter_(1, order, sorted_p)
    return dict(probs=p)


def exact(case, seed):
    if case["kind"] not in ("append", "attend", "probs"):
        return None     # whole numbers: the plain form's are the definition's
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "probs": _exact_probs}[case["kind"]](st, case)
