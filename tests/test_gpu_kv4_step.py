"""A speculative step over the 4-bit cache as a whole, and what its calls do at
its edges: streams without work, refused reservations, calls on other streams."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import E, _cache, _dev, _error, _i32, ctx  # noqa: F401

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
