"""The 4-bit cache and draft verification without a GPU: host checks of
arguments come before any CUDA call, and the layout of a unit (32 positions of
one kv head) covers its bytes exactly once."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "qora-tts-12hz-1.7b_b200")

INVALID, SHAPE, UNSUPPORTED = 1, 2, 6


@pytest.fixture(scope="module")
def lib():
    import qora_b200
    return qora_b200._lib.load()


def test_null_arguments_are_refused(lib):
    one = C.c_void_p(16)          # never dereferenced: the refusal comes first
    out = C.c_void_p()
    assert lib.qora_kv4_create(None, 1, 2, 1, 64, 64, 1, 32, 4, C.byref(out)) == INVALID
    assert lib.qora_kv4_reset(None, None, 0, None) == INVALID
    assert lib.qora_kv4_lengths_host(None, one, None) == INVALID
    assert lib.qora_kv4_state(None, None, None, None) == INVALID
    assert lib.qora_kv4_reserve(None, one, 4, one, one, one, None) == INVALID
    assert lib.qora_kv4_advance(None, one, None) == INVALID
    assert lib.qora_kv4_append(None, 0, one, one, one, one, one, 8, one, one, 1, one, None) == INVALID
    assert lib.qora_kv4_write(None, 0, one, 1, one, one, None) == INVALID
    assert lib.qora_kv4_read(None, 0, one, 1, one, one, None) == INVALID
    assert lib.qora_kv4_attend(None, 0, one, one, 1, 1, one, None) == INVALID
    lib.qora_kv4_destroy(None)


def test_sampling_refusals_come_before_any_cuda_call(lib):
    from qora_b200 import _lib
    one, ctx = C.c_void_p(16), C.create_string_buffer(256)   # a zeroed stand-in: only its address is looked at
    P = _lib.SampleParams
    bad = [(P(0.9, 50, 1.0, 1.05), 0, 8, INVALID), (P(0.9, 50, 1.0, 1.05), 4, 0, INVALID),
           (P(0.9, 50, 1.0, 1.05), 1, 327681, UNSUPPORTED), (P(0.9, 1025, 1.0, 1.0), 1, 4096, UNSUPPORTED),
           (P(0.9, 0, 0.9, 1.0), 1, 4096, UNSUPPORTED), (P(0.9, 4096, 0.9, 1.0), 1, 4096, UNSUPPORTED)]
    for params, B, V, want in bad:
        assert lib.qora_sample_probs(ctx, one, B, V, None, 0, C.byref(params), one, None) == want
    ok = P(0.9, 50, 1.0, 1.05)
    assert lib.qora_sample_probs(ctx, one, 1, 8, None, 3, C.byref(ok), one, None) == INVALID
    assert lib.qora_sample_probs(None, one, 1, 8, None, 0, C.byref(ok), one, None) == INVALID
    v = lib.qora_verify_drafts
    assert v(None, one, one, one, None, one, 1, 1, 8, one, one, None) == INVALID
    assert v(ctx, None, one, one, None, one, 1, 1, 8, one, one, None) == INVALID
    assert v(ctx, one, one, None, None, one, 1, 1, 8, one, one, None) == INVALID
    assert v(ctx, one, one, one, None, one, 0, 1, 8, one, one, None) == INVALID
    assert v(ctx, one, one, one, None, one, 1, -1, 8, one, one, None) == INVALID
    assert v(ctx, one, one, one, None, one, 1, 1, 0, one, one, None) == INVALID
    for K, V in ((1, 2 ** 30 + 1), (1, 2 ** 31 - 1), (2 ** 20 + 1, 8), (2 ** 31 - 1, 1)):
        assert v(ctx, one, one, one, None, one, 1, K, V, one, one, None) == UNSUPPORTED


def test_cache_shapes_are_refused(lib):
    ctx, out = C.create_string_buffer(256), C.c_void_p()

    def create(layers=1, heads=4, kvh=2, hd=64, max_pos=256, streams=2, page=32, pool=8):
        return lib.qora_kv4_create(ctx, layers, heads, kvh, hd, max_pos, streams, page, pool, C.byref(out))
    assert create(layers=0) == INVALID and create(pool=0) == INVALID and create(streams=0) == INVALID
    assert create(hd=96) == UNSUPPORTED and create(heads=3) == SHAPE
    assert create(page=16) == INVALID and create(page=48) == INVALID
    assert create(streams=4097) == UNSUPPORTED and create(max_pos=(1 << 20) + 1) == UNSUPPORTED
    assert create(page=1 << 12, pool=1 << 19) == UNSUPPORTED and create(pool=(1 << 20) + 1) == UNSUPPORTED


def test_unit_layout_covers_every_byte_once(tmp_path):
    """Compiles the layout's functions for the host: each nibble of K and V and
    each scale has its own place, and together they fill 36 * head_dim bytes."""
    src, exe = tmp_path / "probe.cu", tmp_path / "probe"
    src.write_text(r'''
#include "kv4.cuh"
#include <cstdio>
using namespace qora;
template <int D> void show() {
    using U = Kv4Unit<D>;
    for (int r = 0; r < 32; r++) {
        for (int d = 0; d < D; d++)
            printf("%d K %d %d\nN %d V %d %d\n", D, U::k_word(r, d) * 2 + (d & 7), 0, D, U::v_half(r, d) * 2 + (d & 3), 0);
        for (int c = 0; c < D / 32; c++) printf("%d s %d %d\n", D, U::k_scale(r, c), U::v_scale(r, c));
    }
}
int main() { show<64>(); show<128>(); return 0; }
''')
    subprocess.run(["nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(PKG, "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.replace("\nN ", "\n").splitlines()
    for D in (64, 128):
        hit = np.zeros(36 * D * 2, int)
        for line in lines:
            d, what, a, b = line.split()
            if int(d) != D:
                continue
            if what == "s":
                for at in (int(a), int(b)):
                    hit[at * 2:at * 2 + 4] += 1
            else:
                hit[int(a)] += 1
        assert (hit == 1).all()


def test_accept_refuses_null_arguments(lib):
    one = C.c_void_p(16)
    assert lib.qora_kv4_accept(None, one, one, None) == INVALID
    assert lib.qora_kv4_accept(one, None, one, None) == INVALID
    assert lib.qora_kv4_accept(one, one, None, None) == INVALID


def test_writing_what_was_read_keeps_scales_from_2_to_the_minus_21():
    """By the definition: code 7 is used, so amax / 7 of what is held is the scale again.
    Below 2^-21 f16 has fewer than 3 bits for a scale, and that no longer holds."""
    import kv4_ref as R
    rng = np.random.default_rng(0)
    changed = 0
    for e in range(-26, 20):
        x = (2.0 ** e * 7 * np.exp2(rng.random((3000, 1))) * rng.uniform(-1, 1, (3000, 32))).astype(np.float32)
        codes, scales = R.quantise(x)
        again, scales2 = R.quantise(R.held(x))
        moved = (codes != again).any(-1) | (scales != scales2)
        assert not moved[scales >= 2.0 ** -21].any()
        changed += int(moved.sum())
    assert changed > 0
