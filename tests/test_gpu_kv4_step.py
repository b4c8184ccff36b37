"""A speculative step over the 4-bit cache as a whole, and what its calls do at
its edges: streams without work, refused reservations, calls on other streams, one
captured graph from block tables to lengths, and attention against the f32 cache's."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import E, _cache, _dev, _error, _i32, _weights, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

OOM, RANGE = 4, 5


# ------------------------------------------------------------ streams without work
def test_verify_count_of_an_idle_stream(E, ctx):  # noqa: F811
    """Count -1: no token at all, and no error; the streams around it are as without it."""
    rng = np.random.default_rng(3)
    for B, K, V in ((3, 2, 40), (5, 4, 9001), (2, 1, 100000)):
        p = rng.random((B, K + 1, V)).astype(np.float32)
        p /= p.sum(-1, keepdims=True)
        drafts = rng.integers(0, V, (B, K)).astype(np.int32)
        u = rng.random((B, K + 1)).astype(np.float32)
        counts = np.full(B, K, np.int32)
        counts[1] = -1
        bad = p.copy()
        bad[1], drafts[1] = np.nan, -7                      # an idle stream's rows are not read
        for q in (None, np.ascontiguousarray(bad[:, :K])):
            tokens, n_out = E.verify_drafts(ctx, _dev(drafts), None if q is None else _dev(q), _dev(bad), _dev(u), _dev(counts))
            assert _error(ctx) == 0
            tokens, n_out = tokens.cpu().numpy(), n_out.cpu().numpy()
            assert n_out[1] == 0 and (tokens[1] == -1).all()
            for b in range(B):
                if b != 1:
                    want = R.verify(drafts[b], None if q is None else q[b], p[b], u[b], K)
                    assert tokens[b].tolist() == want + [-1] * (K + 1 - len(want)) and n_out[b] == len(want)


def test_advance_within_what_was_reserved(ctx):  # noqa: F811
    """With reserve's offsets, a stream moves by at most the tokens that it was given:
    none for one without tokens, none for all after a refusal, whatever n_out says."""
    kv = _cache(ctx, 1, 2, 1, 64, 256, 4, 32, 8)
    _, _, offsets = kv.reserve(_i32([5, 0, 31, 40]), 100)
    kv.advance(_i32([3, 1, 31, 50]), offsets=offsets)
    assert list(kv.lengths()) == [3, 0, 31, 40] and _error(ctx) == 0
    _, _, offsets = kv.reserve(_i32([1, 0, 200, 1]), 300)   # the pool has 4 pages left
    assert _error(ctx) == OOM
    kv.advance(_i32([1, 1, 5, 1]), offsets=offsets)
    assert list(kv.lengths()) == [3, 0, 31, 40] and _error(ctx) == 0
    _, _, offsets = kv.reserve(_i32([1, 0, 1, 1]), 3)       # and the cache goes on
    kv.advance(_i32([1, 1, -4, 0]), offsets=offsets)                # rolling back stays possible
    assert list(kv.lengths()) == [4, 0, 27, 40] and _error(ctx) == 0


# ------------------------------------------------------------ results on other streams
def _late(stream, n, dtype):
    """Work on `stream` that is still to come, which writes blocks of n values that the
    allocator has back already."""
    import torch
    with torch.cuda.stream(stream):
        blocks = [torch.empty(n, dtype=dtype, device="cuda") for _ in range(64)]
        torch.cuda._sleep(100_000_000)                      # some 0.05 s
        for t in blocks:
            t.fill_(77)


@pytest.mark.parametrize("what", ["reserve", "append", "read", "attend", "probs", "verify"])
def test_results_of_a_call_on_another_stream(E, ctx, orc, what):  # noqa: F811
    """`stream=` without `out`: what the current stream still has to do (writes to memory
    that was freed there, or a fill of the result) does not reach the result."""
    import torch
    heads, kvh, hd, n = 4, 2, 64, 32
    kv = _cache(ctx, 1, heads, kvh, hd, 256, 1, 32, 8)
    qn, kn, cos, sin = (_dev(t) for t in _weights(orc, hd, 3))
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(n, (heads + 2 * kvh) * hd, generator=g, device="cuda")
    counts = _i32([n])
    slots, positions, offsets = kv.reserve(counts, n)
    q = kv.append(0, qkv, qn, kn, cos, sin, positions, slots)
    logits, u = torch.randn(n, 500, generator=g, device="cuda"), torch.rand(n, 3, generator=g, device="cuda")
    target = torch.softmax(torch.randn(n, 3, 500, generator=g, device="cuda"), -1)
    drafts = _i32(np.arange(2 * n).reshape(n, 2))
    calls = {"reserve": (lambda **kw: kv.reserve(counts, n, **kw), [(n, torch.int32), (n, torch.int32), (2, torch.int32)]),
             "append": (lambda **kw: kv.append(0, qkv, qn, kn, cos, sin, positions, slots, **kw), [(n * heads * hd, torch.float32)]),
             "read": (lambda **kw: kv.read(0, slots, **kw), [(n * kvh * hd, torch.float32)] * 2),
             "attend": (lambda **kw: kv.attend(0, q, offsets, n, **kw), [(n * heads * hd, torch.float32)]),
             "probs": (lambda **kw: E.sample_probs(ctx, logits, None, E.default_params(), **kw), [(n * 500, torch.float32)]),
             "verify": (lambda **kw: E.verify_drafts(ctx, drafts, None, target, u, **kw), [(n * 3, torch.int32), (n, torch.int32)])}
    call, blocks = calls[what]
    want = call()
    want = [t.clone() for t in (want if isinstance(want, tuple) else (want,))]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for size, dtype in blocks:
        _late(torch.cuda.current_stream(), size, dtype)
    got = call(stream=side)
    got = got if isinstance(got, tuple) else (got,)
    torch.cuda.synchronize()
    assert _error(ctx) == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------------------ a step in one graph
def test_captured_step_from_tables_to_lengths(E, ctx, orc):  # noqa: F811
    """reserve, append, attend, the logits' rows by stream, the distribution, verification
    and advance in one graph without a return to the host: ragged drafts, streams that
    come and go, a step that the pool refuses.  Replays equal eager calls with the
    counts known on the host, and verification's definition."""
    import torch
    heads, kvh, hd, S, K, V, rows, pool = 4, 2, 64, 4, 3, 200, 18, 10
    qn, kn, cos, sin = (_dev(t) for t in _weights(orc, hd, 4))
    g = torch.Generator(device="cuda").manual_seed(9)
    params = E._lib.SampleParams(0.9, 40, 0.95, 1.1)
    rng = np.random.default_rng(12)

    def inputs(drafted):
        return (_i32(drafted), torch.randn(rows, (heads + 2 * kvh) * hd, generator=g, device="cuda"),
                _i32(rng.integers(0, V, (S, K))), torch.rand(S, K + 1, generator=g, device="cuda"),
                _i32(rng.integers(0, V, (S, K + 1, 8))))

    def program(kv, drafted, qkv, drafts, u, prev, keep):
        counts = drafted + 1                                # tokens: the last one said, and the drafts; -1: idle
        slots, positions, offsets = kv.reserve(counts, rows)
        q = kv.append(0, qkv, qn, kn, cos, sin, positions, slots, out=keep["q"])
        o = kv.attend(0, q, offsets, K + 1, out=keep["o"])
        logits = 30.0 * o[:, :V]
        # row (b, j) is token j of stream b, its last one where it has fewer
        at = torch.minimum(offsets[:-1, None] + torch.arange(K + 1, device="cuda"), offsets[1:, None] - 1)
        dense = logits[at.clamp(min=0).reshape(-1)]
        p = E.sample_probs(ctx, dense, prev.view(S * (K + 1), -1), params).view(S, K + 1, V)
        tokens, n_out = E.verify_drafts(ctx, drafts, None, p, u, drafted)
        kv.advance(n_out, offsets=offsets)
        keep["p"].copy_(p), keep["tokens"].copy_(tokens), keep["n_out"].copy_(n_out)

    def buffers():
        return dict(q=torch.zeros(rows, heads * hd, device="cuda"), o=torch.zeros(rows, heads * hd, device="cuda"),
                    p=torch.zeros(S, K + 1, V, device="cuda"), tokens=_i32(np.zeros((S, K + 1))), n_out=_i32(np.zeros(S)))

    # idle streams, all drafts, none; and a step of all drafts that the pool refuses
    steps = [inputs(d) for d in ([3, -1, 0, 2], [0, 3, -1, 3], [-1, -1, -1, -1], [2, 2, 2, 2], [-1, 0, 3, 1])]
    full = inputs([3, 3, 3, 3])
    kv, eager = (_cache(ctx, 1, heads, kvh, hd, 256, S, 32, pool) for _ in range(2))
    for c in (kv, eager):
        c.reserve(_i32([30, 0, 31, 60]), 121)               # (positions that hold zeros)
        c.advance(_i32([30, 0, 31, 60]))
    bufs, static = buffers(), [t.clone() for t in full]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        program(kv, *static, bufs)
    lens = [30, 0, 31, 60]
    assert list(kv.lengths()) == lens
    for step in steps:
        ref = buffers()
        program(eager, *step, ref)
        for a, b in zip(static, step):
            a.copy_(b)
        for t in bufs.values():
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert _error(ctx) == 0
        drafted, _, drafts, u, _ = (t.cpu().numpy() for t in step)
        for name in ("tokens", "n_out", "q", "o", "p"):
            assert torch.equal(bufs[name], ref[name]), name
        tokens, n_out, p = (bufs[n].cpu().numpy() for n in ("tokens", "n_out", "p"))
        for b in range(S):
            want = [] if drafted[b] < 0 else R.verify(drafts[b], None, p[b], u[b], drafted[b])
            assert tokens[b].tolist() == want + [-1] * (K + 1 - len(want)) and n_out[b] == len(want)
            lens[b] += len(want)
        assert list(kv.lengths()) == list(eager.lengths()) == lens
    # a step that the pool refuses: stream 3 has all the other pages, in full
    held = kv.state()["table"]
    used = {int(held[b, j]) for b in range(3) for j in range(-(-lens[b] // 32))}
    rest = [p for p in range(pool) if p not in used]
    kv.advance(_i32([0, 0, 0, 32 * len(rest) - lens[3]]))
    held[3, :len(rest)] = _i32(rest)
    lens[3] = 32 * len(rest)
    for a, b in zip(static, full):
        a.copy_(b)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert _error(ctx) == OOM and list(kv.lengths()) == lens
    kv.advance(_i32([0, 0, 0, -100]))
    graph.replay()                                          # with pages again it goes on
    torch.cuda.synchronize()
    assert _error(ctx) == 0 and all(a > b for a, b in zip(kv.lengths(), lens[:3]))


# ------------------------------------------------------------ a large cache with little work
@pytest.mark.parametrize("streams,count", [(64, 1), (64, 2), (300, 2)])
def test_attend_goes_by_the_streams_with_tokens(ctx, streams, count):  # noqa: F811
    """One stream's call of a token or two in a cache of many: the work is split as in a cache of one, so
    the bits are the same."""
    import torch
    heads, kvh, hd, length, page = 16, 8, 128, 5000, 64
    pool = -(-(length + count) // page)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(length + count, kvh * hd, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(count, heads * hd, generator=g, device="cuda")
    got = []
    for S, b in ((1, 0), (streams, streams - 3)):
        kv = _cache(ctx, 1, heads, kvh, hd, pool * page, S, page, pool)
        n = np.zeros(S, np.int32)
        n[b] = length
        slots, _, _ = kv.reserve(_i32(n), length)
        kv.write(0, slots, k[:length], v[:length])
        kv.advance(_i32(n))
        n[b] = count
        slots, _, offsets = kv.reserve(_i32(n), count)
        kv.write(0, slots, k[length:], v[length:])
        got.append(kv.attend(0, q, offsets, count))
    assert _error(ctx) == 0 and torch.equal(*got)


# ------------------------------------------------------------ small values
@pytest.mark.parametrize("hd", [64, 128])
def test_writing_what_was_read_at_the_smallest_scales(ctx, hd):  # noqa: F811
    """From 2^-21 on the same codes and scales; below, what the definition gives for the
    values that were read."""
    rng = np.random.default_rng(hd)
    kvh, n = 2, 64
    kv = _cache(ctx, 2, 2, kvh, hd, 64, 1, 32, 2)
    size = 2.0 ** rng.integers(-26, -12, (n, kvh, hd // 32, 1)) * 7
    x = [(size * rng.uniform(-1, 1, (n, kvh, hd // 32, 32))).astype(np.float32).reshape(n, -1) for _ in range(2)]
    slots = _i32(rng.permutation(64))
    kv.write(0, slots, *map(_dev, x))
    once = kv.read(0, slots)
    kv.write(1, slots, *once)
    twice = kv.read(1, slots)
    for src, a, b in zip(x, once, twice):
        a, b = a.cpu().numpy(), b.cpu().numpy()
        rows = lambda t: t.reshape(n, kvh, hd)  # noqa: E731
        assert np.array_equal(rows(a), R.held(rows(src))) and np.array_equal(rows(b), R.held(rows(a)))
        keep = R.quantise(rows(src))[1] >= 2.0 ** -21
        assert np.array_equal(a.reshape(n, kvh, -1, 32)[keep], b.reshape(n, kvh, -1, 32)[keep]) and not np.array_equal(a, b)
    assert _error(ctx) == 0


# ------------------------------------------------------------ the largest cache
def test_reserve_over_the_largest_pool(ctx):  # noqa: F811
    """2^20 pages and 4096 streams: the widest cluster with as much shared memory as a call takes."""
    S, page, pool, max_pos = 4096, 32, 1 << 20, 1 << 14
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 8000, S)
    counts = rng.integers(0, 70, S)
    kv = _cache(ctx, 1, 1, 1, 64, max_pos, S, page, pool)
    keep = -(-lens // page)
    table = np.full((S, max_pos // page), -1, np.int32)
    order = rng.permutation(pool)[:int(keep.sum())]
    table[np.arange(table.shape[1]) < keep[:, None]] = order
    st = kv.state()
    st["table"].copy_(_i32(table))
    st["lengths"].copy_(_i32(lens))
    tokens = int(counts.sum()) + 9
    got = kv.reserve(_i32(counts), tokens)
    assert _error(ctx) == 0
    want = R.reserve(table, lens, counts, page, pool, max_pos, tokens)
    for x, y in zip((st["table"],) + tuple(got), want):
        assert np.array_equal(x.cpu().numpy(), y)


# ------------------------------------------------------------ against the f32 cache
@pytest.mark.parametrize("heads,kvh,hd,length", [(4, 2, 128, 0), (16, 8, 128, 333), (4, 4, 64, 70), (8, 2, 64, 31)])
def test_attend_agrees_with_the_f32_cache(E, ctx, orc, heads, kvh, hd, length):  # noqa: F811
    """qora_kv_attend and qora_kv4_attend over the same keys and values: the f32 slab
    holds what the 4-bit rows stand for, and the new token's own row is one that 4 bits
    hold exactly (a key norm of zeros, values of whole codes)."""
    import torch
    from qora_b200 import _lib
    from qora_b200.engine import _device_view
    rng = np.random.default_rng(hd + length)
    S, max_pos = 2, 512
    qn, _, cos, sin = (_dev(t) for t in _weights(orc, hd, 6))
    kn = torch.zeros(hd, dtype=torch.float16, device="cuda")
    kv4 = _cache(ctx, 1, heads, kvh, hd, max_pos, S, 32, 2 * max_pos // 32)
    slots, _, _ = kv4.reserve(_i32([length + 1] * S), S * (length + 1))
    k, v = (_dev(rng.standard_normal((S * (length + 1), kvh * hd)).astype(np.float32)) for _ in range(2))
    kv4.write(0, slots, k, v)
    kv4.advance(_i32([length] * S))
    k, v = (t.view(S, length + 1, kvh, hd).transpose(1, 2) for t in kv4.read(0, slots))
    kv = E.KvCache(ctx, 1, kvh, hd, max_pos, S)
    ptr = [C.c_void_p() for _ in range(3)]
    _lib.call("qora_kv_layer_ptrs", kv.h, 0, *(C.byref(p) for p in ptr))
    for p, rows in zip(ptr, (k, v)):
        _device_view(p.value, (S, kvh, max_pos, hd), "<f4", "cuda:0", kv)[:, :, :length] = rows[:, :, :length]
    _device_view(ptr[2].value, (S,), "<i4", "cuda:0", kv).fill_(length)
    qkv = _dev(rng.standard_normal((S, (heads + 2 * kvh) * hd)).astype(np.float32))
    codes = rng.integers(-7, 8, (S, kvh * hd // 32, 32))
    codes[..., 5] = 7
    qkv[:, -kvh * hd:] = _dev((codes * 0.25).astype(np.float32).reshape(S, -1))
    positions = _i32([length] * S)
    full = kv.attend(0, qkv, heads, qn.view(torch.int16), kn.view(torch.int16), cos, sin, positions)
    slots, positions, offsets = kv4.reserve(_i32([1] * S), S)
    q = kv4.append(0, qkv, qn, kn, cos, sin, positions, slots)
    mine = kv4.attend(0, q, offsets, 1)
    assert _error(ctx) == 0
    # Each is within its own bound of the definition: kv4_ref.attend's for the 4-bit
    # kernel; for f32 a score's head_dim products and sums, 2^-24 of its sum of
    # magnitudes each, two roundings of q before, twice that for a probability, and 2^-19
    # with 2^-24 a position for exponentials and sums.
    kk, vv = kv4.read(0, slots)
    for b in range(S):
        ks = np.concatenate([k[b, :, :length].transpose(0, 1).cpu().numpy(), kk[b].view(1, kvh, hd).cpu().numpy()])
        vs = np.concatenate([v[b, :, :length].transpose(0, 1).cpu().numpy(), vv[b].view(1, kvh, hd).cpu().numpy()])
        qs = q[b].view(1, heads, hd).cpu().numpy()
        ref, bound = R.attend(qs, ks, vs, length, heads, kvh)
        size = max(np.abs(ks[:, h * kvh // heads]).dot(np.abs(qs[0, h])).max() for h in range(heads)) / np.sqrt(hd)
        wide = (2 * (hd + 16) * 2.0 ** -24 * size + 2.0 ** -19 + (length + 1) * 2.0 ** -24) * np.abs(vs).max()
        a, f = (t[b].view(1, heads, hd).cpu().numpy() for t in (mine, full))
        assert np.all(np.abs(a - ref) <= bound) and np.all(np.abs(a - f) <= bound + wide)
