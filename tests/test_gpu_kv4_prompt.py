"""The prompt kernel of attention over the 4-bit cache (k_kv4_prompt), and the
other beside it: every test here asserts first which kernel its call reaches, by
the rule that qora_kv4_attend chooses by."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import E, _cache, _check, _dev, _error, _filled, _i32, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


def prompt_runs(heads, kvh, hd, streams, tokens, max_count):
    """Whether qora_kv4_attend takes the prompt kernel (prompt_pays, csrc/kv4_attend.cu)."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    G, S = heads // kvh, min(streams, tokens)
    if G * max_count <= 24:
        return False
    rows = G * min(tokens, S * max_count)
    tiles8, tiles128 = kvh * max(S, -(-rows // 8)), kvh * max(S, -(-rows // 128))
    return tiles8 > (600 if hd == 64 else 400) * -(-tiles128 // sms)


@pytest.mark.parametrize("heads,kvh,hd,n", [(8, 1, 128, 416), (8, 1, 64, 640)])
def test_sums_over_a_long_cache(ctx, heads, kvh, hd, n):  # noqa: F811
    """33000 positions, one key far above all others, which are equal, and equal values:
    every probability behind the first is the same number, so additions to a running
    sum round in one direction.  The result is the value itself, whatever the scores.

    The sums of O are added in f32 once in 64 positions, 2^-24 of the sum at most each
    time; the denominator, the products' own additions and the split of P are 2^-19."""
    length, page = 32768, 1024
    assert prompt_runs(heads, kvh, hd, 1, n, n)
    total = length + n
    pool = -(-total // page)
    kv = _cache(ctx, 1, heads, kvh, hd, total, 1, page, pool)
    slots, _, _ = kv.reserve(_i32([total]), total)
    k = np.full((total, kvh * hd), 7 * 0.0625, np.float32)
    k[0] = 7 * 0.125
    v = np.full((total, kvh * hd), 7 * 0.21875, np.float32)
    kv.write(0, slots, _dev(k), _dev(v))
    kv.advance(_i32([length]))
    # scores of position 0 lie d in base 2 above the others: 1.1 to 9.9
    d = np.linspace(1.1, 9.9, n * heads).reshape(n, heads, 1)
    a = d * np.log(2) / (np.sqrt(hd) * 7 * 0.0625)
    q = np.broadcast_to(a, (n, heads, hd)).astype(np.float32).reshape(n, -1)
    out = kv.attend(0, _dev(q), _i32([0, n]), n).cpu().numpy()
    assert _error(ctx) == 0
    worst = float(np.abs(out / np.float32(7 * 0.21875) - 1).max())
    assert worst <= total / 64 * 2.0 ** -24 + 2.0 ** -19, worst


@pytest.mark.parametrize("heads,kvh,hd,lens,counts,most", [
    (4, 2, 64, [37, 0, 90], [2, 3, 1], 3), (16, 8, 128, [37, 0, 90], [2, 3, 1], 3),
    (32, 8, 128, [37, 0, 90], [50, 64, 20], 64), (32, 8, 64, [37, 0, 90], [70, 64, 40], 70)])
def test_nan_values_reach_rows_that_hardly_weigh_them(ctx, heads, kvh, hd, lens, counts, most):  # noqa: F811
    """A NaN value is in the sum whatever its weight, 0 by underflow included, in a
    stream's last unit of positions as in any other."""
    import torch
    page, S = 64, len(lens)
    prompt_case = most > 3
    assert prompt_runs(heads, kvh, hd, S, sum(counts), most) == prompt_case
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 97)
    table, n = kv.state()["table"].cpu().numpy(), sum(counts)
    slot = lambda b, p: int(table[b, p // page]) * page + p % page  # noqa: E731
    # the stream's first key is far above that of the position with the NaN
    top, low = _i32([slot(2, 0)]), 88                        # 88: the last unit holds positions 64 on
    k, v = kv.read(1, top)
    kv.write(1, top, torch.full_like(k, 40.0), v)
    at = _i32([slot(2, low)])
    k, v = kv.read(1, at)
    half = v.clone()
    half[:, :32] = float("nan")
    kv.write(1, at, torch.full_like(k, -40.0), half)
    q = np.abs(rng.standard_normal((n, heads, hd))).astype(np.float32) + 0.5
    got = kv.attend(1, _dev(q.reshape(n, -1)), offsets, most)
    nan = torch.isnan(got).view(n, heads, hd).cpu().numpy()
    want = np.zeros_like(nan)
    want[n - counts[2]:, :heads // kvh, :32] = True
    assert np.array_equal(nan, want) and _error(ctx) == 0


# heads, kv heads, head_dim, page, lengths, new tokens, max_count: streams of one, several
# and no row tiles of 128, of 1, 2, 3, 4 and more key tiles of 64
UNDERSTATED = [
    (32, 8, 128, 32, [70, 0, 161, 5], [200, 40, 40, 40], 32),
    (32, 8, 128, 64, [0, 30, 0, 400], [90, 200, 0, 180], 33),
    (32, 8, 64, 64, [70, 0, 161, 5], [200, 40, 40, 40], 40),
    (24, 8, 64, 32, [3, 64, 129], [260, 130, 2], 90),
]


@pytest.mark.parametrize("heads,kvh,hd,page,lens,counts,most", UNDERSTATED)
def test_a_block_takes_further_row_tiles(ctx, heads, kvh, hd, page, lens, counts, most):  # noqa: F811
    """max_count below the tokens of some streams: the grid has fewer row tiles than
    they have, so blocks take several in turn."""
    assert prompt_runs(heads, kvh, hd, len(lens), sum(counts), most) and heads // kvh * max(counts) > 128
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 90 + hd)
    q = (1.5 * rng.standard_normal((sum(counts), heads, hd))).astype(np.float32)
    got = _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, most)
    # a row's result does not depend on which block takes its tile, nor on the time
    assert prompt_runs(heads, kvh, hd, len(lens), sum(counts), max(counts))
    for mc in (most, max(counts)):
        again = _check(kv, q, offsets, held, lens, counts, heads, kvh, hd, mc)
        assert np.array_equal(again.view(np.uint32), got.view(np.uint32))
    assert _error(ctx) == 0


@pytest.mark.parametrize("heads,kvh,hd,page,lens,counts", [(32, 8, 64, 32, [3, 0, 70], [90, 70, 11]),
                                                          (16, 16, 128, 64, [200, 7], [129, 90])])
def test_captured_prompt_of_many_rows_replays(ctx, heads, kvh, hd, page, lens, counts):  # noqa: F811
    """Lengths, offsets and tables are read at each replay; on a stream of its own beside
    a prompt of another cache."""
    import torch
    n, most = sum(counts), max(counts)
    assert prompt_runs(heads, kvh, hd, len(lens), n, most)
    kv, offsets, held, rng = _filled(ctx, lens, counts, heads, kvh, hd, page, 95)
    other, offsets2, _, _ = _filled(ctx, lens, counts, heads, kvh, hd, page, 96)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    qd, out, side = _dev(q.reshape(n, -1)), torch.zeros(n, heads * hd, device="cuda"), torch.cuda.Stream()
    want = other.attend(1, qd, offsets2, most)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kv.attend(1, qd, offsets, most, out=out)
    for now in (counts, [c // 3 for c in counts], [0] * (len(counts) - 1) + [1]):
        offsets.copy_(_i32(np.concatenate([[0], np.cumsum(now)])))
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        beside = other.attend(1, qd, offsets2, most)
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


def test_prompts_on_two_streams_beside_drafts(ctx):  # noqa: F811
    """Two caches' prompts, of head_dim 64 and 128, and a third's drafts at the same time."""
    import torch
    shapes = [((32, 8, 64, 64), [70, 0], [90, 80], 90), ((32, 8, 128, 32), [5, 33, 90], [60, 50, 40], 60),
              ((32, 8, 128, 64), [900, 33, 0, 5], [5, 0, 3, 6], 6)]
    jobs = []
    for i, (shape, lens, counts, most) in enumerate(shapes):
        assert prompt_runs(*shape[:3], len(lens), sum(counts), most) == (i < 2)
        kv, offsets, held, rng = _filled(ctx, lens, counts, *shape, 100 + i)
        q = _dev(rng.standard_normal((sum(counts), shape[0] * shape[2])).astype(np.float32))
        jobs.append((kv, q, offsets, most, kv.attend(1, q, offsets, most), torch.zeros_like(q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for kv, q, offsets, most, want, out, s in jobs:
            with torch.cuda.stream(s):
                kv.attend(1, q, offsets, most, out=out)
    torch.cuda.synchronize()
    for kv, q, offsets, most, want, out, s in jobs:
        assert bool((out == want).all())
    assert _error(ctx) == 0
