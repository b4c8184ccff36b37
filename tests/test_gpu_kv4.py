"""The 4-bit paged KV cache (qora_kv4) on the GPU against float64 restatements
(tests/kv4_ref.py): block tables, append, plain writes and reads, attention."""
import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu

INVALID, OOM, RANGE, UNSUPPORTED = 1, 4, 5, 6


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


def _cache(ctx, *a, **kw):
    from qora_b200.kv4 import Kv4Cache
    return Kv4Cache(ctx, *a, **kw)


def _dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t.to(dtype) if dtype is not None else t).cuda()


def _i32(a):
    return _dev(np.asarray(a, np.int32))


def _error(ctx):
    """Status of the device error flag (cleared)."""
    from qora_b200 import _lib
    try:
        ctx.check_device_error()
    except _lib.QoraError as e:
        return e.status
    return 0


# ------------------------------------------------------------ block tables
@pytest.mark.parametrize("page,lens,counts,spare", [
    (32, [0], [1], 0),                                     # the first token of all
    (32, [31, 32, 33, 0], [1, 1, 1, 0], 0),                # page borders; a stream without tokens
    (64, [0, 5, 64, 127, 128, 200], [64, 0, 65, 1, 300, 57], 3),
    (32, [0] * 70, [3] * 70, 1),
    (128, [1000, 0, 257], [0, 0, 0], 2),                   # nothing new
    (32, list(range(0, 1500, 11)), [i % 7 for i in range(137)], 5),
])
def test_reserve_matches_definition(ctx, page, lens, counts, spare):
    S, max_pos = len(lens), 2048
    rng = np.random.default_rng(S + page)
    keep = [-(-n // page) for n in lens]
    need = sum(-(-(n + c) // page) for n, c in zip(lens, counts))
    pool = need + spare
    per = max_pos // page
    order = iter(rng.permutation(pool))
    table = np.full((S, per), -1, np.int32)
    for b in range(S):
        for j in range(keep[b]):
            table[b, j] = next(order)
    kv = _cache(ctx, 1, 2, 1, 64, max_pos, S, page, pool)
    st = kv.state()
    st["table"].copy_(_i32(table))
    st["lengths"].copy_(_i32(lens))
    max_tokens = sum(counts) + 3
    want = R.reserve(table, lens, counts, page, pool, max_pos, max_tokens)
    for _ in range(2):                                      # a second call gives the same
        got = kv.reserve(_i32(counts), max_tokens)
        assert _error(ctx) == 0
        for x, y in zip((st["table"],) + tuple(got), want):
            assert np.array_equal(x.cpu().numpy(), y)
    kv.advance(_i32(counts))
    assert list(kv.lengths()) == [a + b for a, b in zip(lens, counts)]
    assert _error(ctx) == 0


@pytest.mark.parametrize("why,counts,max_tokens,status", [
    ("pool", [200, 10, 200], 600, OOM), ("tokens", [3, 3, 3], 8, RANGE), ("length", [0, 1000, 0], 2000, RANGE),
    ("negative", [1, -1, 1], 16, RANGE), ("overflow", [2 ** 31 - 1, 2 ** 31 - 1, 5], 16, RANGE)])
def test_reserve_refuses_as_a_whole(ctx, why, counts, max_tokens, status):
    kv = _cache(ctx, 1, 2, 1, 64, 512, 3, 32, 10)
    st = kv.state()
    kv.reserve(_i32([33, 0, 5]), 64)
    kv.advance(_i32([33, 0, 5]))
    before = st["table"].clone()
    assert _error(ctx) == 0
    slots, positions, offsets = kv.reserve(_i32(counts), max_tokens)
    assert _error(ctx) == status
    assert (slots == -1).all() and (positions == 0).all() and (offsets == 0).all()
    assert bool((st["table"] == before).all()) and list(kv.lengths()) == [33, 0, 5]
    kv.reserve(_i32([1, 1, 1]), 3)                          # the cache goes on
    assert _error(ctx) == 0


def test_reserve_counts_past_31_bits(ctx):
    """4096 streams that share one page of 2^20 positions (their tables say so)
    ask for all the rest of it: 2^32 - 4096 tokens, and no new page."""
    S, P = 4096, 1 << 20
    kv = _cache(ctx, 1, 1, 1, 64, P, S, P, 1)
    st = kv.state()
    st["table"].zero_()
    st["lengths"].fill_(1)
    slots, positions, offsets = kv.reserve(_i32([P - 1] * S), 100)
    assert _error(ctx) == RANGE
    assert (slots == -1).all() and (positions == 0).all() and (offsets == 0).all()
    slots, positions, offsets = kv.reserve(_i32([1] + [0] * (S - 2) + [1]), 2)
    assert _error(ctx) == 0 and slots.tolist() == [1, 1] and positions.tolist() == [1, 1]
    p = slots.data_ptr()
    assert kv._L.qora_kv4_reserve(kv.h, p, 2 ** 30 + 1, p, p, p, None) == UNSUPPORTED    # refused before any access


def test_bad_table_entry_is_an_error_not_an_access(ctx):
    import torch
    kv = _cache(ctx, 1, 2, 1, 64, 128, 2, 32, 6)
    kv.reserve(_i32([40, 3]), 43)
    kv.advance(_i32([40, 3]))
    st = kv.state()
    st["table"][0, 1] = 6                                   # one past the pool
    kv.reserve(_i32([1, 1]), 2)
    assert _error(ctx) == RANGE
    out = kv.attend(0, torch.zeros(2, 128, device="cuda"), _i32([0, 1, 2]), 1)
    assert _error(ctx) == RANGE and out.shape == (2, 128)
    st["table"][0, 1] = -1
    kv.attend(0, torch.zeros(2, 128, device="cuda"), _i32([0, 1, 2]), 1)
    assert _error(ctx) == RANGE


def test_rolled_back_pages_are_free_again(ctx):
    kv = _cache(ctx, 1, 2, 1, 64, 256, 2, 32, 4)
    kv.reserve(_i32([96, 32]), 128)
    kv.advance(_i32([96, 32]))
    kv.reserve(_i32([0, 1]), 1)
    assert _error(ctx) == OOM
    kv.advance(_i32([-40, 0]))                              # 56 positions: two pages
    slots, _, _ = kv.reserve(_i32([0, 1]), 1)
    assert _error(ctx) == 0 and int(slots[0]) // 32 == 2
    kv.advance(_i32([-57, 0]))                              # past zero
    assert _error(ctx) == RANGE and list(kv.lengths()) == [0, 32]
    kv.reset([1])
    assert list(kv.lengths()) == [0, 0]
    kv.reserve(_i32([128, 0]), 128)
    assert _error(ctx) == 0


def test_state_views_keep_the_cache(ctx):
    import gc
    import weakref
    kv = _cache(ctx, 1, 2, 1, 64, 64, 2, 32, 4)
    alive, table = weakref.ref(kv), kv.state()["table"]
    del kv
    gc.collect()
    assert alive() is not None and bool((table == -1).all())
    row = table[0]
    del table
    gc.collect()
    assert alive() is not None and bool((row == -1).all())
    del row
    gc.collect()
    assert alive() is None


# ------------------------------------------------------------ rows
def _weights(orc, hd, seed):
    rng = np.random.default_rng(seed)
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2))
    cos, sin = (t.reshape(-1, hd // 2) for t in orc.rope_tables(hd, 512, 1e6))
    return qn, kn, cos, sin


@pytest.mark.parametrize("heads,kvh,hd,page,n", [(16, 8, 128, 64, 5), (4, 2, 64, 32, 33), (3, 3, 128, 32, 1),
                                                 (8, 1, 64, 128, 70), (16, 8, 128, 32, 150)])
def test_append_matches_definition(ctx, orc, heads, kvh, hd, page, n):
    import torch
    rng = np.random.default_rng(hd + n)
    layers, layer, pool = 3, 1, -(-n // page) + 2
    qn, kn, cos, sin = _weights(orc, hd, n)
    kv = _cache(ctx, layers, heads, kvh, hd, pool * page, 1, page, pool)
    qkv = (rng.standard_normal((n, (heads + 2 * kvh) * hd)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32)
    qkv[0, -hd:] = 0.0                                     # a value row of zeros
    qkv[n // 2, -32:] = np.arange(32) * 0.5 - 7.0          # ties: scale 1.0 (amax / 7 = 8.5 / 7 ... -7 / 7)
    qkv[n // 2, -1] = 7.0
    qkv[n // 2, -32:-1] = np.clip(qkv[n // 2, -32:-1], -6.5, 6.5)
    pos = rng.integers(0, 512, n).astype(np.int32)
    slots = rng.permutation(pool * page)[:n].astype(np.int32)
    args = [_dev(qn), _dev(kn), _dev(cos), _dev(sin), _i32(pos), _i32(slots)]
    q = kv.append(layer, _dev(qkv), *args)
    k, v = kv.read(layer, args[-1])
    assert _error(ctx) == 0
    rq, rk, rv = R.append(qkv, heads, kvh, hd, qn, kn, cos, sin, pos)
    # q in f32.  With u = 2^-24: the sum of squares is off by 8 u (8 products and sums
    # in a lane, 4 exchanges, all terms positive, less than 12 roundings of which the
    # square root halves the effect: 6 u), the mean, eps, root and quotient by 4 u more
    # (half of the first two), x inv gamma by 2 u, and the rotation a c - b s by 2 u of
    # |a c| + |b s|: 14 u of that sum covers it.  (When q was computed in f64 this
    # was one rounding; the reference's own rows are f32 arithmetic.)
    a = np.stack([[R.norm_rope(qkv[i, h * hd:(h + 1) * hd], qn, np.ones(hd // 2), np.zeros(hd // 2))
                   for h in range(heads)] for i in range(n)])
    c, s = np.abs(cos[pos])[:, None], np.abs(sin[pos])[:, None]
    one, two = np.abs(a[..., :hd // 2]), np.abs(a[..., hd // 2:])
    size = np.concatenate([one * c + two * s, two * c + one * s], -1).reshape(n, -1)
    assert np.all(np.abs(q.cpu().numpy() - rq) <= 14 * 2.0 ** -24 * size + 1e-12)
    assert np.array_equal(k.cpu().numpy(), rk) and np.array_equal(v.cpu().numpy(), rv)
    # the other layers and the other slots were left as they were (zeros)
    rest = _i32(np.setdiff1d(np.arange(pool * page), slots))
    for lay, sl in ((0, args[-1]), (2, args[-1]), (layer, rest)):
        assert not any(bool(t.any()) for t in kv.read(lay, sl))
    # a half-tie goes to the even code
    assert float(v[n // 2, -31]) in (-6.0, -7.0) and bool(torch.isfinite(v).all())


def test_rows_behind_the_last_token_are_left(ctx, orc):
    import torch
    heads, kvh, hd, n = 4, 2, 64, 6
    qn, kn, cos, sin = _weights(orc, hd, 1)
    kv = _cache(ctx, 1, heads, kvh, hd, 64, 1, 32, 2)
    qkv = torch.randn(n, (heads + 2 * kvh) * hd, device="cuda")
    q = torch.full((n, heads * hd), 7.0, device="cuda")
    slots = _i32([0, 1, -1, -1, 5, -1])
    kv.append(0, qkv, _dev(qn), _dev(kn), _dev(cos), _dev(sin), _i32([0, 1, 9999, -5, 2, 3]), slots, out=q)
    assert _error(ctx) == 0
    assert bool((q[[2, 3, 5]] == 7.0).all()) and bool((q[[0, 1, 4]] != 7.0).all())
    k = torch.full((n, kvh * hd), 3.0, device="cuda")
    v = torch.full((n, kvh * hd), 3.0, device="cuda")
    kv.read(0, slots, out=(k, v))
    assert bool((k[[2, 3, 5]] == 3.0).all()) and bool((v[[2, 3, 5]] == 3.0).all())
    # no rows at all
    kv.append(0, qkv[:0], _dev(qn), _dev(kn), _dev(cos), _dev(sin), _i32([]), _i32([]))
    assert _error(ctx) == 0


@pytest.mark.parametrize("slot,pos", [(64, 0), (-2, 0), (3, 512), (3, -1), (2 ** 31 - 1, 0)])
def test_append_outside_pool_or_table_is_an_error(ctx, orc, slot, pos):
    import torch
    heads, kvh, hd = 4, 2, 64
    qn, kn, cos, sin = _weights(orc, hd, 1)
    kv = _cache(ctx, 1, heads, kvh, hd, 64, 1, 32, 2)
    qkv = torch.ones(2, (heads + 2 * kvh) * hd, device="cuda")
    kv.append(0, qkv, _dev(qn), _dev(kn), _dev(cos), _dev(sin), _i32([0, pos]), _i32([1, slot]))
    assert _error(ctx) == RANGE
    k, _ = kv.read(0, _i32(range(64)))
    assert sorted(set(torch.nonzero(k.any(-1))[:, 0].tolist())) == [1]


@pytest.mark.parametrize("hd", [64, 128])
def test_write_then_read_then_write_keeps_codes(ctx, hd):
    import torch
    rng = np.random.default_rng(hd)
    kvh, n = 3, 64
    kv = _cache(ctx, 2, 3, kvh, hd, 128, 1, 32, 4)
    x = rng.standard_normal((2, n, kvh, hd)).astype(np.float32)
    x[0] *= np.float32(1e-3)
    x[1, 3] *= np.float32(1e9)          # past f16's scales: saturates
    x[1, 4] = 1e-9                      # under f16's smallest: zeros
    x[0, 5, 1, 7] = np.nan              # the group reads back as NaN
    x[0, 6, 1, 40] = np.inf
    slots = _i32(rng.permutation(128)[:n])
    kv.write(1, slots, _dev(x[0].reshape(n, -1)), _dev(x[1].reshape(n, -1)))
    k, v = kv.read(1, slots)
    assert _error(ctx) == 0
    for got, src in ((k, x[0]), (v, x[1])):
        want = R.held(src).reshape(n, -1)
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    assert int(torch.isnan(k).sum()) == 64 and float(v.view(n, kvh, hd)[3].abs().max()) == 7 * 65504
    kv.write(0, slots, k, v)
    k2, v2 = kv.read(0, slots)
    assert np.array_equal(k.cpu().numpy(), k2.cpu().numpy(), equal_nan=True) and bool((v == v2).all())


# ------------------------------------------------------------ attention
def _filled(ctx, lens, counts, heads, kvh, hd, page, seed, k_size=1.0, v_size=1.0, spare=1):
    """A cache whose streams hold lens positions and counts new ones, with what
    they hold: kv, offsets, [(k, v) per stream]."""
    rng = np.random.default_rng(seed)
    S = len(lens)
    pool = sum(-(-(a + b) // page) for a, b in zip(lens, counts)) + spare
    kv = _cache(ctx, 2, heads, kvh, hd, max(a + b for a, b in zip(lens, counts)) + 5, S, page, pool)
    rows = []
    for step in (lens, counts):
        slots, positions, offsets = kv.reserve(_i32(step), sum(step) + 1)
        n = sum(step)
        k = (k_size * rng.standard_normal((n + 1, kvh, hd))).astype(np.float32)
        v = (v_size * (rng.standard_normal((n + 1, kvh, hd)) + 0.3)).astype(np.float32)
        kv.write(1, slots, _dev(k.reshape(n + 1, -1)), _dev(v.reshape(n + 1, -1)))
        rows.append((R.held(k), R.held(v), np.concatenate([[0], np.cumsum(step)])))
        if step is lens:
            kv.advance(_i32(lens))
    assert _error(ctx) == 0
    held = []
    for b in range(S):
        held.append([np.concatenate([part[i][part[2][b]:part[2][b + 1]] for part in rows]) for i in (0, 1)])
    return kv, offsets, held, rng


def _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, max_count, out=None):
    got = kv.attend(1, _dev(q.reshape(q.shape[0], -1)), offsets, max_count, out=out).cpu().numpy()
    at = 0
    worst = 0.0
    for b, (n, c) in enumerate(zip(lens, counts)):
        if c:
            ref, bound = R.attend(q[at:at + c], held[b][0], held[b][1], n, heads, kvh)
            err = np.abs(got[at:at + c].reshape(c, heads, hd) - ref)
            assert np.isfinite(got[at:at + c]).all()
            worst = max(worst, float((err / bound).max()))
        at += c
    assert worst <= 1.0, worst
    return got


CASES = [
    # heads, kvh, hd, page, lengths, new tokens
    (16, 8, 128, 64, [0], [1]),
    (16, 8, 128, 64, [700], [1]),
    (4, 2, 64, 32, [31, 32, 33, 95, 0], [1, 1, 1, 1, 1]),
    (16, 8, 128, 32, [0, 1, 30, 64, 500, 3], [5, 0, 4, 1, 6, 2]),
    (4, 4, 64, 64, [100, 0, 7], [3, 4, 1]),
    (8, 1, 128, 128, [200, 13], [1, 3]),
    (6, 2, 64, 32, [65, 129], [2, 7]),
    (32, 8, 128, 64, [1000], [1]),
    (4, 2, 128, 32, [0, 17], [70, 33]),                     # prompts
    (16, 8, 128, 64, [0, 100], [129, 64]),
    (6, 2, 64, 32, [40, 0, 3], [200, 1, 43]),
    (2, 2, 128, 64, [300], [257]),
    (16, 8, 64, 64, [5] * 40, [1] * 40),
    (2, 1, 128, 32, [0, 0, 0], [0, 1, 0]),
    (16, 8, 128, 64, [2500, 40, 0], [1, 1, 1]),
    (32, 8, 128, 32, [40, 0, 7, 65] * 4, [8, 7, 8, 8] * 4),  # few rows of many streams: the prompt kernel
    (32, 8, 64, 64, [40, 0, 7, 65] * 9, [7, 8, 0, 8] * 9),
]


@pytest.mark.parametrize("heads,kvh,hd,page,lens,counts", CASES)
def test_attend_matches_definition(ctx, heads, kvh, hd, page, lens, counts):
    import torch
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, len(lens) + hd)
    n = sum(counts)
    q = (1.5 * rng.standard_normal((n + 2, heads, hd))).astype(np.float32)
    out = torch.full((n + 2, heads * hd), 9.0, device="cuda")
    got = _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, max(counts), out)
    assert (got[n:] == 9.0).all()                           # rows behind the last token
    # whichever kernel max_count chooses, and again: the same call gives the same bits
    again = kv.attend(1, _dev(q.reshape(n + 2, -1)), offsets, max(counts)).cpu().numpy()
    assert np.array_equal(got[:n].view(np.uint32), again[:n].view(np.uint32))
    for other in (1, 2, 4, 8, 100):
        _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, other)
    assert _error(ctx) == 0


@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-30, 1.0, 1.0), (3e4, 1e-3, 1e-4), (1e6, 1e-5, 3e5), (30.0, 1.0, 1e-6)])
def test_attend_any_range(ctx, q_size, k_size, v_size):
    lens, counts, heads, kvh, hd = [150, 3], [1, 2], 4, 2, 128
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, 32, 5, k_size, v_size)
    q = (q_size * rng.standard_normal((3, heads, hd))).astype(np.float32)
    for mc in (1, 2, 64):                                   # each of the kernels
        _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, mc)
    assert _error(ctx) == 0


def test_attend_sees_nothing_behind_the_last_position(ctx):
    """Rows behind a stream's end hold NaN and infinities: the results do not change."""
    import torch
    lens, counts, heads, kvh, hd, page = [37, 0, 90], [2, 3, 1], 4, 2, 64, 64
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 3)
    table = kv.state()["table"].cpu().numpy()
    behind = [int(table[b, p // page]) * page + p % page for b in range(3)
              for p in range(lens[b] + counts[b], -(-(lens[b] + counts[b]) // page) * page)]
    bad = torch.full((len(behind), kvh * hd), float("nan"), device="cuda")
    kv.write(1, _i32(behind), bad, bad)
    q = rng.standard_normal((6, heads, hd)).astype(np.float32)
    for mc in (1, 8, 64):
        _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, mc)
    # within a stream a NaN reaches the tokens that see it, and only those
    at = _i32([int(table[1, 0]) * page + 1])
    k, v = kv.read(1, at)
    half = v.clone()
    half[:, :32] = float("nan")                             # one scale group of the first kv head
    for keys, values in ((k * float("nan"), v), (k, v * float("nan")), (k, half)):
        kv.write(1, at, keys, values)
        for mc in (1, 3, 64):
            out = kv.attend(1, _dev(q.reshape(6, -1)), offsets, mc)
            nan = torch.isnan(out).any(-1).cpu().numpy()
            assert list(nan) == [False, False, False, True, True, False]
            if values is half:
                first = torch.isnan(out[3:5].view(2, heads, hd))
                assert bool(first[:, :2, :32].all()) and int(first.sum()) == 2 * 2 * 32
    q[0, 1, 3] = np.inf
    for mc in (1, 3, 64):
        out = kv.attend(1, _dev(q.reshape(6, -1)), offsets, mc).view(6, heads, hd)
        assert bool(torch.isnan(out[0, 1]).all()) and bool(torch.isfinite(out[0, 0]).all())
    assert _error(ctx) == 0


@pytest.mark.parametrize("hd,lens,counts", [(64, [37, 0, 90], [2, 3, 1]), (128, [0, 161, 5], [1, 2, 70])])
def test_what_a_page_held_before_does_not_matter(ctx, hd, lens, counts):
    """The largest finite scales behind the streams' ends, as pages of other streams
    may leave them: the same bits as behind zeros, small values and all."""
    import torch
    heads, kvh, page = 4, 2, 64
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 31, 1e-3, 1e-4)
    table = kv.state()["table"].cpu().numpy()
    behind = _i32([int(table[b, p // page]) * page + p % page for b in range(3)
                   for p in range(lens[b] + counts[b], -(-(lens[b] + counts[b]) // page) * page)])
    n = sum(counts)
    q = (50.0 * rng.standard_normal((n, heads, hd))).astype(np.float32)
    for mc in (1, 8, 64):
        got = []
        for size in (0.0, 1e30):
            rows = torch.full((behind.numel(), kvh * hd), size, device="cuda")
            kv.write(1, behind, rows, rows)
            got.append(_check(kv, q, offsets, held, lens, counts, heads, kvh, hd, mc))
        assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
    assert _error(ctx) == 0


# Shapes with rows enough for the prompt kernel: 400 (head_dim 64: 600) tiles of 8 rows.
MANY = [(32, 8, 128, 32, [37, 0, 90, 161], [50, 31, 1, 47]), (32, 16, 64, 64, [100, 5, 0], [90, 77, 0]),
        (30, 10, 128, 64, [64, 0], [33, 100]), (16, 16, 128, 32, [3, 200], [129, 100])]


@pytest.mark.parametrize("heads,kvh,hd,page,lens,counts", MANY)
@pytest.mark.parametrize("q_size,k_size,v_size", [(1.5, 1.0, 1.0), (1e-30, 1.0, 1.0), (3e4, 1e-3, 1e-4), (1e6, 1e-5, 3e5)])
def test_many_rows_any_range(ctx, heads, kvh, hd, page, lens, counts, q_size, k_size, v_size):
    import torch
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 60 + hd, k_size, v_size)
    n = sum(counts)
    q = (q_size * rng.standard_normal((n + 3, heads, hd))).astype(np.float32)
    out = torch.full((n + 3, heads * hd), 9.0, device="cuda")
    got = _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, max(counts), out)
    assert (got[n:] == 9.0).all()
    assert np.array_equal(_check(kv, q, offsets, held, lens, counts, heads, kvh, hd, max(counts))[:n], got[:n])
    _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, 1)    # (the other kernel)
    assert _error(ctx) == 0


@pytest.mark.parametrize("heads,kvh,hd,page,lens,counts", MANY)
def test_many_rows_see_nothing_behind_and_nan_where_it_is(ctx, heads, kvh, hd, page, lens, counts):
    """Behind the streams' ends: zeros, the largest scales and NaN give the same bits.  A
    NaN inside reaches the rows that see it, in its scale group for values."""
    import torch
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 70, 1e-3, 1e-4)
    table, S, n, most = kv.state()["table"].cpu().numpy(), len(lens), sum(counts), max(counts)
    slot = lambda b, p: int(table[b, p // page]) * page + p % page
    behind = _i32([slot(b, p) for b in range(S) for p in range(lens[b] + counts[b], -(-(lens[b] + counts[b]) // page) * page)])
    q = (50.0 * rng.standard_normal((n, heads, hd))).astype(np.float32)
    got = []
    for size in (0.0, 1e30, float("nan")):
        rows = torch.full((behind.numel(), kvh * hd), size, device="cuda")
        kv.write(1, behind, rows, rows)
        got.append(_check(kv, q, offsets, held, lens, counts, heads, kvh, hd, most))
    assert all(np.array_equal(g, got[0]) for g in got)
    first = lens[0] + 20                                     # tokens 20 on of stream 0 see it
    at = _i32([slot(0, first)])
    k, v = kv.read(1, at)
    half = v.clone()
    half[:, hd - 32:hd] = float("nan")                       # the first kv head's last group
    for keys, values in ((k * float("nan"), v), (k, v * float("nan")), (k, half)):
        kv.write(1, at, keys, values)
        nan = torch.isnan(kv.attend(1, _dev(q.reshape(n, -1)), offsets, most)).view(n, heads, hd).cpu().numpy()
        want = np.zeros_like(nan)
        want[20:counts[0], :heads // kvh if values is half else heads, hd - 32 if values is half else 0:] = True
        assert np.array_equal(nan, want)
    kv.write(1, at, k, v)
    q[2, 1, 3] = np.inf
    nan = torch.isnan(kv.attend(1, _dev(q.reshape(n, -1)), offsets, most)).view(n, heads, hd)
    assert bool(nan[2, 1].all()) and int(nan.sum()) == hd
    assert _error(ctx) == 0


def test_captured_many_rows_replay_with_other_lengths(ctx):
    import torch
    heads, kvh, hd, page, lens, counts = 32, 8, 128, 32, [37, 0, 90], [50, 64, 20]
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 80)
    n = sum(counts)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    qd, out, side = _dev(q.reshape(n, -1)), torch.zeros(n, heads * hd, device="cuda"), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kv.attend(1, qd, offsets, 64, out=out)
    other = _filled(ctx, lens, counts, heads, kvh, hd, page, 81)
    want = other[0].attend(1, qd, other[1], 64)
    torch.cuda.synchronize()
    for now in (counts, [3, 64, 0], [0, 0, 1], [0, 0, 0]):
        offsets.copy_(_i32(np.concatenate([[0], np.cumsum(now)])))
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()                                   # and another cache's prompt beside it
        beside = other[0].attend(1, qd, other[1], 64)
        torch.cuda.synchronize()
        assert bool((beside == want).all())
        got, at = out.cpu().numpy(), 0
        for b, c in enumerate(now):
            if c:
                ref, bound = R.attend(q[at:at + c], held[b][0][:lens[b] + c], held[b][1][:lens[b] + c], lens[b], heads, kvh)
                assert np.all(np.abs(got[at:at + c].reshape(c, heads, hd) - ref) <= bound)
            at += c
        assert (got[at:] == 7.0).all()
    assert _error(ctx) == 0


def test_unaligned_pointers_are_refused(ctx, orc):
    import torch
    from qora_b200 import _lib
    heads, kvh, hd = 4, 2, 64
    qn, kn, cos, sin = (_dev(t) for t in _weights(orc, hd, 1))
    kv = _cache(ctx, 1, heads, kvh, hd, 64, 1, 32, 2)
    wide = torch.zeros(1 + 2 * (heads + 2 * kvh) * hd, device="cuda")[1:].view(2, -1)
    narrow = torch.zeros(1 + 2 * kvh * hd, device="cuda")[1:].view(2, -1)
    i = _i32([0, 1])
    for call in (lambda: kv.append(0, wide, qn, kn, cos, sin, i, i), lambda: kv.write(0, i, narrow, narrow),
                 lambda: kv.read(0, i, out=(narrow, narrow)),
                 lambda: kv.attend(0, wide.view(-1)[:2 * heads * hd].view(2, -1), i, 1)):
        with pytest.raises(_lib.QoraError) as e:
            call()
        assert e.value.status == INVALID
    assert _error(ctx) == 0


def test_attend_refuses(ctx):
    import torch
    from qora_b200 import _lib
    kv = _cache(ctx, 1, 4, 2, 64, 64, 2, 32, 4)
    q = torch.zeros(3, 256, device="cuda")
    with pytest.raises(_lib.QoraError):
        kv.attend(1, q, _i32([0, 1, 2]), 1)                 # layer
    with pytest.raises(_lib.QoraError):
        kv.attend(0, q, _i32([0, 1, 2]), 0)                 # max_count
    with pytest.raises(ValueError):
        kv.attend(0, q, _i32([0, 1]), 1)                    # offsets too short
    with pytest.raises(ValueError):
        kv.attend(0, q.double(), _i32([0, 1, 2]), 1)
    with pytest.raises(ValueError):
        kv.reserve(_i32([1]), 4)
    with pytest.raises(ValueError):
        kv.reserve(torch.zeros(2, dtype=torch.int64, device="cuda"), 4)
    assert _error(ctx) == 0
    out = torch.full((3, 256), 5.0, device="cuda")
    for offsets in ([0, 4, 4], [2, 1, 3], [-1, 0, 1], [0, 1, 70]):   # rows that are not there, falling, negative, past the cache
        kv.attend(0, q, _i32(offsets), 1, out=out)
        assert _error(ctx) == RANGE
    kv.state()["lengths"][0] = 65
    out.fill_(5.0)
    kv.attend(0, q, _i32([0, 1, 2]), 1, out=out)            # a length past the cache: its row is skipped
    assert _error(ctx) == RANGE
    assert bool((out[[0, 2]] == 5.0).all())


def test_captured_step_replays_with_other_lengths(ctx, orc):
    """reserve + append + attend + advance in one CUDA graph on its own stream:
    replays take the lengths and counts of their time, and equal eager calls."""
    import torch
    heads, kvh, hd, S, rows = 4, 2, 64, 3, 12
    qn, kn, cos, sin = _weights(orc, hd, 4)
    w = [_dev(qn), _dev(kn), _dev(cos), _dev(sin)]
    rng = np.random.default_rng(8)
    steps = [([3, 0, 4], None), ([1, 1, 1], None), ([4, 4, 4], None), ([0, 0, 0], None), ([2, 3, 1], None)]
    steps = [(c, rng.standard_normal((rows, (heads + 2 * kvh) * hd)).astype(np.float32)) for c, _ in steps]

    def program(kv, counts, qkv, out):
        slots, positions, offsets = kv.reserve(counts, rows)
        q = kv.append(0, qkv, *w, positions, slots)
        kv.attend(0, q, offsets, 4, out=out)
        kv.advance(counts)

    eager = _cache(ctx, 1, heads, kvh, hd, 64, S, 32, 6)
    want = []
    for c, x in steps:
        out = torch.zeros(rows, heads * hd, device="cuda")
        program(eager, _i32(c), _dev(x), out)
        want.append(out.cpu().numpy())
    kv = _cache(ctx, 1, heads, kvh, hd, 64, S, 32, 6)
    counts, qkv = _i32([0, 0, 0]), torch.zeros(rows, (heads + 2 * kvh) * hd, device="cuda")
    out = torch.zeros(rows, heads * hd, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        program(kv, counts, qkv, out)
    for (c, x), ref in zip(steps, want):
        counts.copy_(_i32(c))
        qkv.copy_(_dev(x))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy()[:sum(c)], ref[:sum(c)])
        assert not out[sum(c):].any()
    assert _error(ctx) == 0 and list(kv.lengths()) == list(eager.lengths())


def test_two_streams_and_a_replayed_graph(ctx):
    """Prompts on one cache, drafts on another and a captured step of a third, each on
    a stream of its own at the same time: the bits of one after the other."""
    import torch
    shapes = [([70, 0], [150, 200], 64), ([900, 33, 0, 5], [5, 0, 3, 6], 6), ([400] * 9, [1] * 9, 1)]
    jobs = []
    for i, (lens, counts, most) in enumerate(shapes):
        kv, offsets, held, rng = _filled(ctx, lens, counts, 4, 2, 128, 64, 40 + i)
        q = _dev(rng.standard_normal((sum(counts), 4 * 128)).astype(np.float32))
        jobs.append((kv, q, offsets, most, kv.attend(1, q, offsets, most), torch.zeros_like(q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    kv, q, offsets, most, _, out, s = jobs[2]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for _ in range(3):
            kv.attend(1, q, offsets, most, out=out)
    for _ in range(20):
        for kv, q, offsets, most, want, out, s in jobs[:2]:
            with torch.cuda.stream(s):
                kv.attend(1, q, offsets, most, out=out)
        with torch.cuda.stream(jobs[2][6]):
            graph.replay()
    torch.cuda.synchronize()
    for kv, q, offsets, most, want, out, s in jobs:
        assert bool((out == want).all())
    assert _error(ctx) == 0


def test_captured_prompt_replays(ctx):
    """A prompt's attention in a graph reads lengths, offsets and tables at each replay."""
    import torch
    lens, counts, heads, kvh, hd = [3, 0], [90, 40], 4, 2, 64
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, 32, 50)
    q = rng.standard_normal((130, heads, hd)).astype(np.float32)
    qd, out = _dev(q.reshape(130, -1)), torch.zeros(130, heads * hd, device="cuda")
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        kv.attend(1, qd, offsets, 90, out=out)
    for counts in ([90, 40], [17, 40], [0, 1]):
        held_now = [[x[:n + c] for x in h] for h, n, c in zip(held, lens, counts)]
        offsets.copy_(_i32([0, counts[0], sum(counts)]))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got, at = out.cpu().numpy(), 0
        for b, c in enumerate(counts):
            if c:
                ref, bound = R.attend(q[at:at + c], *held_now[b], lens[b], heads, kvh)
                assert np.all(np.abs(got[at:at + c].reshape(c, heads, hd) - ref) <= bound)
            at += c
        assert (got[at:] == 7.0).all()
    assert _error(ctx) == 0


def test_long_cache_past_32_bit_offsets(ctx):
    """A pool of more than 2^31 bytes: the stream's pages lie at its end."""
    import torch
    heads, kvh, hd, page = 16, 8, 128, 1024
    layers = 14
    pool = 140                                             # 140 * 14 * 8 * 1024 * 144 B = 2.3 GB
    kv = _cache(ctx, layers, heads, kvh, hd, 4 * page, 1, page, pool)
    st = kv.state()
    st["table"][0, :3] = _i32([pool - 1, pool - 2, pool - 3])
    n = 2 * page + 40
    pos = np.arange(n + 1)
    slots = _i32((pool - 1 - pos // page) * page + pos % page)
    rng = np.random.default_rng(2)
    k, v = (rng.standard_normal((n + 1, kvh, hd)).astype(np.float32) for _ in range(2))
    kv.write(layers - 1, slots, _dev(k.reshape(n + 1, -1)), _dev(v.reshape(n + 1, -1)))
    st["lengths"][0] = n
    q = rng.standard_normal((1, heads, hd)).astype(np.float32)
    got = kv.attend(layers - 1, _dev(q.reshape(1, -1)), _i32([0, 1]), 1).cpu().numpy().reshape(1, heads, hd)
    ref, bound = R.attend(q, R.held(k), R.held(v), n, heads, kvh)
    assert (np.abs(got - ref) <= bound).all()
    assert _error(ctx) == 0
