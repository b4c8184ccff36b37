"""The prompt kernel of attention over the 4-bit cache (k_kv4_prompt), and the
other beside it: every test here asserts first which kernel its call reaches, by
the rule that qora_kv4_attend chooses by."""
import numpy as np
import pytest

from test_gpu_kv4 import E, _cache, _dev, _error, _filled, _i32, ctx  # noqa: F401

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
