"""qora_sample_probs and qora_verify_drafts against float64 restatements
(tests/kv4_ref.py), and a speculative decode of the tiny talker over the 4-bit
cache with all of its operators."""
import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu

INVALID, RANGE, UNSUPPORTED = 1, 5, 6


@pytest.fixture(scope="module")
def E():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("-m gpu tests need a CUDA device")
    from qora_b200 import engine
    return engine


@pytest.fixture(scope="module")
def ctx(E):
    return E.Context(0)


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _error(ctx):
    from qora_b200 import _lib
    try:
        ctx.check_device_error()
    except _lib.QoraError as e:
        return e.status
    return 0


# ------------------------------------------------------------ probabilities
def _check_probs(E, ctx, x, prev, params):
    got = E.sample_probs(ctx, _dev(x), None if prev is None else _dev(prev), E._lib.SampleParams(*params)).cpu().numpy()
    assert _error(ctx) == 0
    for r in range(x.shape[0]):
        ref = R.probs(x[r], None if prev is None else prev[r], params[0], params[1], params[2], params[3])
        # expf is off by 2^-22, its argument (at most the range of z) and the
        # penalty's results by one f32 rounding each, the result by one more
        fin = x[r][np.isfinite(x[r])].astype(np.float64)
        t = params[0] if params[0] > 0 else 1.0
        tol = 2.0 ** -21 + 2.0 ** -23 * (np.abs(fin).max() * 2 * params[3] ** 3) / t
        assert np.all(np.abs(got[r] - ref) <= tol * ref + 1e-38), (r, np.abs(got[r] - ref).max())
    return got


@pytest.mark.parametrize("B,V,params,n_prev", [
    (3, 320, (0.9, 50, 1.0, 1.05), 16), (1, 1, (0.9, 50, 1.0, 1.0), 0), (2, 2, (1.0, 1, 1.0, 1.0), 0),
    (5, 2048, (0.9, 50, 0.9, 1.2), 40), (2, 2047, (1.3, 1024, 0.95, 1.0), 0), (4, 2048, (0.7, 0, 1.0, 1.1), 3),
    (2, 2049, (0.0, 40, 1.0, 1.0), 0), (3, 33, (0.9, 32, 0.5, 1.05), 5), (2, 40, (0.9, 40, 1.0, 1.05), 5),
    (2, 50000, (0.8, 50, 0.95, 1.1), 64), (2, 151936, (0.9, 1000, 0.9, 1.0), 0), (1, 151936, (1.0, 0, 1.0, 1.0), 0),
    (1, 327680, (0.9, 50, 1.0, 1.05), 8)])
def test_probs_match_definition(E, ctx, B, V, params, n_prev):
    rng = np.random.default_rng(V)
    x = (3 * rng.standard_normal((B, V))).astype(np.float32)
    if V > 100:
        x[0, V // 4:V // 4 + 60] = -np.inf                  # forbidden tokens
    prev = None
    if n_prev:
        prev = rng.integers(0, V, (B, n_prev)).astype(np.int32)
        prev[:, 1:3] = prev[:, :1]                          # one token said three times
        prev[:, -1] = x.argmax(-1)
    got = _check_probs(E, ctx, x, prev, params)
    if 0 < params[1] < V:
        assert ((got > 0).sum(-1) <= params[1]).all()


@pytest.mark.parametrize("V", [300, 2048, 5000, 100000])
def test_probs_ties_go_to_the_lowest_index(E, ctx, V):
    """All logits equal, and equal ones around the top-k border: what is kept is
    lowest-index first, however many there are."""
    x = np.zeros((3, V), np.float32)
    x[1, ::7] = 1.0
    x[2] = -np.float32(1e30)
    x[2, V // 2:] = 2.0
    got = _check_probs(E, ctx, x, None, (0.9, 50, 1.0, 1.0))
    assert list(np.nonzero(got[0])[0]) == list(range(50))
    assert set(np.nonzero(got[1])[0]) <= set(range(V)) and (got[1] > 0).sum() == 50
    assert list(np.nonzero(got[2])[0]) == list(range(V // 2, V // 2 + 50))


@pytest.mark.parametrize("V", [257, 1500, 2049, 9001, 20000, 60000])
@pytest.mark.parametrize("top_k", [50, 200, 1000])
@pytest.mark.parametrize("mask", [-1e9, float(np.finfo(np.float32).min)])
def test_probs_of_masked_rows(E, ctx, V, top_k, mask):
    """Most tokens masked by a large negative number: fewer left than top_k, about as
    many, and more, and all but one."""
    rng = np.random.default_rng(V + top_k)
    left = [1, min(V, top_k // 2), min(V, top_k + 1), V // 2]
    x = np.full((len(left), V), mask, np.float32)
    for r, n in enumerate(left):
        at = rng.permutation(V)[:n]
        x[r, at] = (3 * rng.standard_normal(n)).astype(np.float32)
    got = E.sample_probs(ctx, _dev(x), None, E._lib.SampleParams(0.9, top_k, 0.95 if top_k < V else 1.0, 1.0)).cpu().numpy()
    assert _error(ctx) == 0
    for r in range(len(left)):
        ref = R.probs(x[r], None, 0.9, top_k, 0.95 if top_k < V else 1.0, 1.0)
        # as in _check_probs, with the range of the logits that are left (masked ones are 0
        # exactly: e^-1e9); a cut is exact in 64 bits
        tol = 2.0 ** -21 + 2.0 ** -23 * 2 * np.abs(x[r][x[r] > mask]).max() / 0.9
        assert np.array_equal(got[r] > 0, ref > 0)
        assert np.all(np.abs(got[r] - ref) <= tol * ref)


@pytest.mark.parametrize("V", [300, 2048, 5000, 100000])
@pytest.mark.parametrize("top_k", [50, 600])
def test_probs_zeros_of_both_signs_are_equal(E, ctx, V, top_k):
    """Logits of +0 and -0, as masking by a product leaves them, tie: the lower index
    comes first, with all of the row zeros (radix selection) and with few (sorting)."""
    if top_k >= V:
        top_k = V // 2
    rng = np.random.default_rng(V + top_k)
    x = np.zeros((4, V), np.float32)
    x[0, ::2] = -0.0                                        # -0 first of each pair
    x[1, rng.permutation(V)[:V // 2]] = -0.0
    x[2:] = -5.0 - rng.random((2, V)).astype(np.float32)
    zeros = np.sort(rng.permutation(V)[:min(V, top_k + 40)])
    x[2, zeros] = np.where(np.arange(len(zeros)) % 3 == 0, 0.0, -0.0)
    x[3] = x[2]
    x[3, zeros[-10:]] = 1.5                                 # ten above the zeros
    for top_p in (1.0, 0.9):
        got = _check_probs(E, ctx, x, None, (0.9, top_k, top_p, 1.0))
        for r in range(4):
            assert np.array_equal(got[r] > 0, R.probs(x[r], None, 0.9, top_k, top_p, 1.0) > 0)


@pytest.mark.parametrize("V,n_prev", [(300, 3000), (2048, 4096), (50000, 4096), (50001, 777)])
def test_probs_of_a_long_history(E, ctx, V, n_prev):
    """Thousands of mentions, most of a few tokens, some outside the vocabulary."""
    rng = np.random.default_rng(V)
    x = (3 * rng.standard_normal((3, V))).astype(np.float32)
    prev = rng.integers(-5, V + 5, (3, n_prev)).astype(np.int32)
    prev[1, ::2] = 7                                        # one token said n_prev / 2 times
    prev[2, : n_prev // 2] = rng.integers(0, 9, n_prev // 2)
    x[1, 7], x[2, :9] = 2.0, np.linspace(-1, 1, 9)
    penalty = 1.0005                                        # 2000 times: a factor of e
    params = E._lib.SampleParams(0.9, 200, 1.0, penalty)
    got = E.sample_probs(ctx, _dev(x), _dev(prev), params).cpu().numpy()
    assert _error(ctx) == 0
    assert np.array_equal(got, E.sample_probs(ctx, _dev(x), _dev(prev), params).cpu().numpy())
    for r in range(3):
        ref = R.probs(x[r], prev[r], 0.9, 200, 1.0, penalty)
        # an f32 logit after t mentions has t roundings, and the difference of two of them is
        # divided by the temperature; its largest value is 15.  What the roundings may swap at
        # the border of top_k is within that of each other too
        t = np.bincount(prev[r][(prev[r] >= 0) & (prev[r] < V)], minlength=V).max()
        tol = 2.0 ** -21 + 2 * (t + 2) * 2.0 ** -24 * 15 / 0.9
        same = (got[r] > 0) == (ref > 0)
        assert np.all(np.abs(got[r] - ref)[same] <= tol * ref[same] + 1e-38)
        edge = ref[ref > 0].min()
        assert np.all(np.abs(np.maximum(got[r], ref)[~same] - edge) <= 2 * tol * edge)


def test_probs_agree_with_the_sampler(E, ctx):
    """qora_sample draws what the cumulative probabilities give for its random numbers."""
    import torch
    rng = np.random.default_rng(4)
    B, V = 64, 2048
    x = _dev((2 * rng.standard_normal((B, V))).astype(np.float32))
    prev = _dev(rng.integers(0, V, (B, 16)).astype(np.int32))
    params = E.default_params()
    state = rng.integers(1, 2 ** 62, B)
    s = [int(v) for v in state]
    toks = E.sample_token(ctx, x, prev, _dev(state.astype(np.int64)), params).cpu().numpy()
    p = E.sample_probs(ctx, x, prev, params).cpu().numpy().astype(np.float64)
    for b in range(B):
        v = s[b]
        v ^= (v << 13) & (2 ** 64 - 1)
        v ^= v >> 7
        v ^= (v << 17) & (2 ** 64 - 1)
        cum = np.cumsum(p[b])
        i = int(np.searchsorted(cum, v / 2 ** 64, side="right"))
        near = np.abs(cum - v / 2 ** 64).min() < 1e-5       # a draw on a border may go either way in f32
        assert near or toks[b] == i
    assert bool(torch.isfinite(x).all())


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("V,top_k", [(500, 50), (500, 0), (60000, 50)])
def test_probs_of_a_bad_row_are_zero_and_an_error(E, ctx, bad, V, top_k):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, V)).astype(np.float32)
    x[1, V - 3] = bad
    got = E.sample_probs(ctx, _dev(x), None, E._lib.SampleParams(1.0, top_k, 1.0, 1.0)).cpu().numpy()
    assert _error(ctx) == INVALID
    assert not got[1].any() and np.allclose(got[[0, 2]].sum(-1), 1.0, atol=1e-5)
    x[1] = -np.inf
    got = E.sample_probs(ctx, _dev(x), None, E._lib.SampleParams(1.0, top_k, 1.0, 1.0)).cpu().numpy()
    assert _error(ctx) == INVALID and not got[1].any()


def test_probs_refuse(E, ctx):
    import torch
    from qora_b200 import _lib
    x = torch.zeros(2, 64, device="cuda")
    with pytest.raises(_lib.QoraError):
        E.sample_probs(ctx, x, None, _lib.SampleParams(1.0, 0, 0.9, 1.0))
    with pytest.raises(ValueError):
        E.sample_probs(ctx, x.double(), None, E.default_params())
    with pytest.raises(ValueError):
        E.sample_probs(ctx, x, torch.zeros(2, 4, device="cuda"), E.default_params())
    with pytest.raises(ValueError):
        E.sample_probs(ctx, x, None, E.default_params(), out=torch.zeros(2, 63, device="cuda"))
    assert _error(ctx) == 0


# ------------------------------------------------------------ verification
def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _check_verify(E, ctx, drafts, q, p, u, counts):
    B, K = drafts.shape
    tokens, n_out = E.verify_drafts(ctx, _dev(drafts), None if q is None else _dev(q), _dev(p), _dev(u),
                                    None if counts is None else _dev(counts))
    tokens, n_out = tokens.cpu().numpy(), n_out.cpu().numpy()
    for b in range(B):
        want = R.verify(drafts[b], None if q is None else q[b], p[b], u[b], K if counts is None else int(counts[b]))
        assert n_out[b] == len(want)
        assert list(tokens[b]) == want + [-1] * (K + 1 - len(want)), b
    return tokens, n_out


@pytest.mark.parametrize("B,K,V,dist", [(1, 1, 1, True), (7, 4, 320, True), (33, 5, 2048, True), (16, 3, 2047, False),
                                        (4, 0, 100, True), (5, 40, 65, True), (3, 2, 8193, True), (4, 3, 50001, True),
                                        (3, 4, 151936, True), (3, 2, 151936, False), (300, 2, 33, True)])
def test_verify_matches_definition(E, ctx, B, K, V, dist):
    rng = np.random.default_rng(B * 1000 + V)
    t = 2 * rng.standard_normal((B, K + 1, V))
    p = _softmax(t)
    q = _softmax(t[:, :K] + 0.7 * rng.standard_normal((B, K, V)))
    drafts = np.array([[rng.choice(V, p=q[b, i].astype(np.float64) / q[b, i].astype(np.float64).sum())
                        for i in range(K)] for b in range(B)], np.int32).reshape(B, K)
    if not dist:
        drafts = p[:, :K].argmax(-1).astype(np.int32)
    u = rng.random((B, K + 1)).astype(np.float32)
    _check_verify(E, ctx, drafts, q if dist else None, p, u, None)
    counts = rng.integers(0, K + 1, B).astype(np.int32)
    _check_verify(E, ctx, drafts, q if dist else None, p, u, counts)
    assert _error(ctx) == 0


def test_verify_edges(E, ctx):
    V, K = 200, 2
    p = np.zeros((8, K + 1, V), np.float32)
    q = np.zeros((8, K, V), np.float32)
    d = np.full((8, K), 3, np.int32)
    u = np.full((8, K + 1), 0.5, np.float32)
    p[:, :, 3] = 1.0
    q[:, :, 3] = 1.0                     # 0: equal one-hot rows: all pass
    p[1, 0], q[1, 0] = 0, 0              # 1: p = q = 0 at the draft, nothing left: token 0
    p[2, 0], q[2, 0] = 1.0 / V, 1.0 / V  # 2: u = 1 rejects an equal pair; the difference is empty: from the target
    u[2, 0] = 1.0
    u[3, K] = 1.0                        # 3: u = 1 draws the last token with weight
    p[3, 2, :] = 0
    p[3, 2, 5:9] = 0.25
    u[4] = 0.0                           # 4: u = 0 accepts, and draws the first token with weight
    p[4, 2, :] = 0
    p[4, 2, 77:80] = 1 / 3
    u[5, 0] = np.nan                     # 5: NaN rejects
    p[5, 0, 9] = 0.5
    p[6, 0, :] = np.nan                  # 6: NaN target: rejected, no weight: token 0
    u[7, K] = np.nan                     # 7: NaN draws as 0
    tokens, n_out = E.verify_drafts(ctx, _dev(d), _dev(q), _dev(p), _dev(u))
    tokens, n_out = tokens.cpu().numpy().tolist(), n_out.cpu().numpy().tolist()
    assert tokens[0] == [3, 3, 3] and tokens[1] == [0, -1, -1]
    assert tokens[2] == [100, -1, -1]
    assert tokens[3] == [3, 3, 8] and tokens[4] == [3, 3, 77]
    assert tokens[5] == [9, -1, -1] and tokens[6] == [0, -1, -1] and tokens[7] == [3, 3, 3]
    assert n_out == [3, 1, 1, 3, 3, 1, 1, 3] and _error(ctx) == 0


def test_verify_out_of_range(E, ctx):
    V, K = 64, 3
    p = np.full((4, K + 1, V), 1.0 / V, np.float32)
    d = np.array([[1, 64, 2], [1, -1, 2], [1, 2, 3], [1, 2, 3]], np.int32)
    u = np.full((4, K + 1), 0.01, np.float32)
    counts = np.array([3, 3, 9, -4], np.int32)
    for q in (p[:, :K].copy(), None):
        tokens, n_out = E.verify_drafts(ctx, _dev(d), None if q is None else _dev(q), _dev(p),
                                        _dev(u * (1.0 if q is not None else 0.1)), _dev(counts))
        assert _error(ctx) == RANGE
        assert n_out.tolist() == [2, 2, 4, 1]
        assert tokens[:2, 0].tolist() == [1, 1] and tokens[2, :3].tolist() == [1, 2, 3]


def test_verify_keeps_the_target_distribution(E, ctx):
    """Frequencies of the first token over 200000 streams: the target's, whatever the
    draft's distribution.  A count of a token with probability p has standard deviation
    sqrt(n p (1 - p)); five of them bound each of 12 tokens."""
    import torch
    B, V = 200000, 12
    rng = np.random.default_rng(0)
    p1, q1 = _softmax(rng.standard_normal(V)), _softmax(1.5 * rng.standard_normal(V))
    g = torch.Generator(device="cuda").manual_seed(3)
    q = _dev(q1).expand(B, 1, V).contiguous()
    p = _dev(p1).expand(B, 2, V).contiguous()
    drafts = torch.multinomial(q[:, 0], 1, generator=g).to(torch.int32)
    tokens, _ = E.verify_drafts(ctx, drafts, q, p, torch.rand(B, 2, generator=g, device="cuda"))
    seen = np.bincount(tokens[:, 0].cpu().numpy(), minlength=V)
    assert np.all(np.abs(seen - B * p1) <= 5 * np.sqrt(B * p1 * (1 - p1)))


def test_verify_refuses(E, ctx):
    import torch
    d = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    p, u = torch.zeros(2, 4, 9, device="cuda"), torch.zeros(2, 4, device="cuda")
    with pytest.raises(ValueError):
        E.verify_drafts(ctx, d, p, p, u)                    # draft_probs of K + 1 rows
    with pytest.raises(ValueError):
        E.verify_drafts(ctx, d, None, p[:, :3], u)
    with pytest.raises(ValueError):
        E.verify_drafts(ctx, d, None, p, u[:, :3])
    with pytest.raises(ValueError):
        E.verify_drafts(ctx, d.long(), None, p, u)
    with pytest.raises(ValueError):
        E.verify_drafts(ctx, d, None, p, u, counts=d[:, 0].float())
    assert _error(ctx) == 0


# ------------------------------------------------------------ all together
class _Talker4:
    """The tiny talker's decoder layers over a 4-bit cache (talker.rs:263-360)."""

    def __init__(self, E, ctx, orc, streams, max_pos=128):
        import qora_b200
        from qora_b200.kv4 import Kv4Cache
        self.E, self.ctx = E, ctx
        self.cfg = c = qora_b200.ModelConfig.tiny()
        self.w = qora_b200.synth_talker(c)
        self.talker = E.Talker(ctx, self.w, max_batch=1)
        q4 = lambda w: E.DeviceQ4(ctx, w)  # noqa: E731
        self.layers = [{n: q4(getattr(L, n)) for n in ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj",
                                                       "up_proj", "down_proj")} |
                       {n: _dev(getattr(L, n).view(np.int16)) for n in ("q_norm", "k_norm", "input_norm",
                                                                        "post_attn_norm")} for L in self.w.layers]
        self.final = _dev(self.w.final_norm.view(np.int16))
        self.head = q4(self.w.codec_head)
        cos, sin = orc.rope_tables(c.t_head_dim, max_pos, c.rope_theta)
        self.cos, self.sin = _dev(cos), _dev(sin)
        self.kv = Kv4Cache(ctx, c.t_layers, c.t_heads, c.t_kv_heads, c.t_head_dim, max_pos, streams, 32,
                           streams * (max_pos // 32))

    def step(self, x, counts, rows, max_count):
        """x [rows][hidden] of the new tokens (rows behind them unused) -> logits [rows][vocab]."""
        import torch
        E = self.E
        slots, positions, offsets = self.kv.reserve(counts, rows)
        for i, L in enumerate(self.layers):
            h = E.rms_norm_f16(self.ctx, x, L["input_norm"])
            qkv = torch.cat([L[n].gemm(h) for n in ("q_proj", "k_proj", "v_proj")], -1).contiguous()
            q = self.kv.append(i, qkv, L["q_norm"], L["k_norm"], self.cos, self.sin, positions, slots)
            o = self.kv.attend(i, q, offsets, max_count, out=torch.zeros_like(q))
            x = x + L["o_proj"].gemm(o)
            h = E.rms_norm_f16(self.ctx, x, L["post_attn_norm"])
            x = x + L["down_proj"].gemm((torch.nn.functional.silu(L["gate_proj"].gemm(h)) * L["up_proj"].gemm(h)).contiguous())
        return self.head.gemm(E.rms_norm_f16(self.ctx, x, self.final))


def test_speculative_decode_equals_plain_decode(E, ctx, orc):
    """Greedy decode of three streams, one token a step, against the same with
    drafted tokens (right ones, wrong ones, fewer for some streams) verified over the
    4-bit cache: the same tokens, with the lengths moved on the device only."""
    import torch
    S, total, K = 3, 24, 4
    greedy = E._lib.SampleParams(1.0, 1, 1.0, 1.0)          # top-1: the distribution is one token

    def embed(m, tokens):
        return m.talker.embed_codec_token(tokens.reshape(-1))

    prompts = [7, 33, 20]
    rng = np.random.default_rng(6)
    toks = [rng.integers(0, 320, n) for n in prompts]

    def prefill(m):
        x = torch.cat([embed(m, torch.from_numpy(t)) for t in toks])
        counts = _dev(np.array(prompts, np.int32))
        logits = m.step(x.contiguous(), counts, sum(prompts), max(prompts))
        m.kv.advance(counts)
        last = torch.from_numpy(np.cumsum(prompts) - 1).cuda()
        return logits[last].contiguous()

    plain = _Talker4(E, ctx, orc, S)
    logits, said = prefill(plain), []
    one = _dev(np.ones(S, np.int32))
    for _ in range(total + K + 1):
        tok = logits.argmax(-1).to(torch.int32)
        said.append(tok)
        logits = plain.step(embed(plain, tok).contiguous(), one, S, 1)
        plain.kv.advance(one)
    said = torch.stack(said, 1).cpu().numpy()               # [S][...]
    assert _error(ctx) == 0

    spec = _Talker4(E, ctx, orc, S)
    logits = prefill(spec)
    out = [[int(t)] for t in logits.argmax(-1)]
    steps = 0
    while min(len(o) for o in out) < total:
        n_draft = rng.integers(0, K + 1, S).astype(np.int32)
        drafts = np.zeros((S, K), np.int32)
        for b in range(S):
            at = len(out[b])
            drafts[b] = said[b, np.minimum(np.arange(at, at + K), said.shape[1] - 1)]
            if rng.random() < 0.5:                          # a wrong draft
                drafts[b, rng.integers(0, K)] += 1
            drafts[b] %= 320
            if at >= total:
                n_draft[b] = 0
        counts = n_draft + 1
        rows = torch.cat([torch.tensor([out[b][-1], *drafts[b, :n_draft[b]]]) for b in range(S)])
        logits = spec.step(embed(spec, rows).contiguous(), _dev(counts), int(counts.sum()), K + 1)
        probs = E.sample_probs(ctx, logits, None, greedy)
        target = torch.zeros(S, K + 1, 320, device="cuda")
        at = 0
        for b in range(S):
            target[b, :counts[b]] = probs[at:at + counts[b]]
            at += counts[b]
        tokens, n_out = E.verify_drafts(ctx, _dev(drafts), None, target, torch.full((S, K + 1), 0.5, device="cuda"), _dev(n_draft))
        spec.kv.advance(n_out)
        for b in range(S):
            out[b] += tokens[b, :int(n_out[b])].tolist()
        steps += 1
        assert _error(ctx) == 0
    assert steps < total
    for b in range(S):
        n = min(len(out[b]), said.shape[1])
        assert out[b][:n] == said[b, :n].tolist(), b
    assert list(spec.kv.lengths()) == [p + len(o) - 1 for p, o in zip(prompts, out)]


def test_4bit_talker_is_near_the_f32_talker(E, ctx, orc):
    """The same prompt through the f32 cache and the 4-bit one.  With keys and values of
    the prompt written back as the 4-bit cache holds them, the f32 path's attention and
    this one agree to the arithmetic (2e-4 of the logits' scale, the tiny model's own
    tolerance); the 4-bit rounding itself is covered by the cache's tests."""
    import torch
    m = _Talker4(E, ctx, orc, 1)
    rng = np.random.default_rng(9)
    x = m.talker.embed_codec_token(torch.from_numpy(rng.integers(0, 320, 12))).contiguous()
    counts = _dev(np.array([12], np.int32))
    logits = m.step(x, counts, 12, 12)
    m.kv.advance(counts)
    kv = m.talker.new_kv(max_pos=64)
    m.talker.prefill_talker_raw_from(x, kv, 0)
    # one step on each with the f32 cache's rows as the 4-bit cache holds them
    slots = _dev(np.arange(12, dtype=np.int32) + int(m.kv.state()["table"][0, 0]) * 32)
    c = m.cfg
    for layer in range(c.t_layers):
        k32, v32 = kv.layer_tensors(layer)
        rows = lambda t: t[0, :, :12].transpose(0, 1).reshape(12, -1).contiguous()  # noqa: E731
        m.kv.write(layer, slots, rows(k32), rows(v32))
        k4, v4 = m.kv.read(layer, slots)
        for mine, full in ((k4, rows(k32)), (v4, rows(v32))):
            # half a step of the largest code, and the scale's own f16 rounding
            g = full.view(12, -1, 32)
            step = g.abs().amax(-1, keepdim=True) / 7
            assert bool(((mine.view_as(g) - g).abs() <= step * (0.5 + 7 * 2.0 ** -11) + 1e-7).all())
    assert logits.shape == (12, 320) and bool(torch.isfinite(logits).all()) and _error(ctx) == 0
