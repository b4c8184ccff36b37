"""Kv4Cache's checks of its arguments, without a GPU: a cache that is not there
(CPU tensors stand for the device's) and entry points that only record that they
were reached."""
import pytest
import torch

H, KV, D, S, PER = 4, 2, 64, 3, 4


@pytest.fixture
def kv():
    from qora_b200.kv4 import Kv4Cache
    kv = object.__new__(Kv4Cache)
    kv.num_heads, kv.kv_heads, kv.head_dim, kv.streams = H, KV, D, S
    kv.device, kv._dev, kv.h, kv.calls = "cpu", -1, None, []
    for name in ("_reserve", "_advance", "_append", "_write", "_read", "_attend", "_accept"):
        setattr(kv, name, lambda *a, name=name: kv.calls.append(name) or 0)
    kv._stream = lambda stream: 0
    return kv


def f32(*shape):
    return torch.zeros(*shape)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def append(kv, n=5, **kw):
    a = dict(qkv=f32(n, (H + 2 * KV) * D), q_norm=torch.zeros(D, dtype=torch.float16),
             k_norm=torch.zeros(D, dtype=torch.float16), rope_cos=f32(16, D // 2), rope_sin=f32(16, D // 2),
             positions=i32(n), slots=i32(n), out=None) | kw
    return kv.append(0, a["qkv"], a["q_norm"], a["k_norm"], a["rope_cos"], a["rope_sin"], a["positions"], a["slots"],
                     out=a["out"])


def test_right_shapes_pass(kv):
    assert append(kv).shape == (5, H * D)
    append(kv, qkv=f32(5, H + 2 * KV, D), slots=i32(9), positions=i32(9), out=f32(8, H * D))
    append(kv, q_norm=torch.zeros(D, dtype=torch.int16), rope_cos=f32(16 * D // 2), rope_sin=f32(16 * D // 2))
    append(kv, 0)
    kv.write(0, i32(5), f32(5, KV * D), f32(7, KV, D))
    kv.write(0, i32(5), f32(5 * KV * D), f32(5, KV * D))
    kv.read(0, i32(5), out=(f32(5, KV, D), f32(9, KV * D)))
    kv.attend(0, f32(5, H, D), i32(S + 1), 2, out=f32(6, H * D))
    kv.reserve(i32(S), 4, out=(i32(4), i32(6), i32(S + 1)))
    kv.advance(i32(S))
    kv.advance(i32(S), offsets=i32(S + 1))
    assert kv.calls == ["_append"] * 4 + ["_write"] * 2 + ["_read", "_attend", "_reserve", "_advance", "_accept"]


@pytest.mark.parametrize("call", [
    lambda kv: append(kv, qkv=f32(5, (H + 2 * KV) * D + 1)),            # wider rows would be misread
    lambda kv: append(kv, qkv=f32(5, (H + 2 * KV) * D * 2)),
    lambda kv: append(kv, out=f32(5, 2 * H * D)),
    lambda kv: append(kv, out=f32(4, H * D)),
    lambda kv: append(kv, rope_cos=f32(16, D), rope_sin=f32(16, D)),    # a table of whole heads
    lambda kv: append(kv, rope_sin=f32(17, D // 2)),
    lambda kv: append(kv, slots=i32(4)),
    lambda kv: append(kv, positions=i32(5).long()),
    lambda kv: kv.write(0, i32(5), f32(5, KV * D + 8), f32(5, KV * D)),
    lambda kv: kv.write(0, i32(5), f32(5, KV * D), f32(5, 2 * KV, D)),
    lambda kv: kv.write(0, i32(5), f32(4, KV * D), f32(5, KV * D)),
    lambda kv: kv.read(0, i32(5), out=(f32(5, KV * D), f32(5, H * D))),
    lambda kv: kv.attend(0, f32(5, (H + 2 * KV) * D), i32(S + 1), 1),   # qkv in place of q
    lambda kv: kv.attend(0, f32(5, H * D), i32(S + 2), 1),
    lambda kv: kv.attend(0, f32(5, H * D), i32(S), 1),
    lambda kv: kv.attend(0, f32(5, H * D), i32(S + 1), 1, out=f32(5, 2 * H * D)),
    lambda kv: kv.attend(0, f32(5, 2 * H * D)[:, ::2], i32(S + 1), 1),
    lambda kv: kv.reserve(i32(S + 1), 4),
    lambda kv: kv.reserve(i32(S), 4, out=(i32(3), i32(4), i32(S + 1))),
    lambda kv: kv.advance(i32(S + 1)),
    lambda kv: kv.advance(i32(S), offsets=i32(S)),
])
def test_wrong_shapes_are_refused(kv, call):
    with pytest.raises(ValueError):
        call(kv)
    assert kv.calls == []


@pytest.mark.parametrize("norm", [torch.zeros(D, dtype=torch.bfloat16), torch.zeros(D), torch.zeros(2, D, dtype=torch.float16),
                                  torch.zeros(2 * D, dtype=torch.float16)[::2], torch.zeros(D // 2, dtype=torch.float16)])
@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
def test_norms_are_f16(kv, name, norm):
    """bf16 has as many bytes, and would be read as other numbers."""
    with pytest.raises(ValueError):
        append(kv, **{name: norm})
    assert kv.calls == []
