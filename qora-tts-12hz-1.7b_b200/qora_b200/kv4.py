"""The 4-bit paged KV cache (qora_kv4): block tables built on the GPU, the
append with qk-norm and rotation, and attention over the cache.

A speculative decode step of every stream, without a return to the host
(drafted: int32 [streams], drafts of each; -1: idle):

    slots, positions, offsets = kv.reserve(drafted + 1, max_tokens)
    for each layer:
        q = kv.append(layer, qkv, q_norm, k_norm, cos, sin, positions, slots)
        o = kv.attend(layer, q, offsets, K + 1)
    # logits are packed by offsets; verification takes K + 1 rows of every stream
    row = torch.minimum(offsets[:-1, None] + torch.arange(K + 1, device=dev), offsets[1:, None] - 1)
    p = engine.sample_probs(ctx, logits[row.clamp(min=0).view(-1)], prev, params)
    tokens, n_out = engine.verify_drafts(ctx, drafts, draft_probs, p.view(streams, K + 1, -1), uniforms, drafted)
    kv.advance(n_out, offsets=offsets)

Tensors are on the context's device and contiguous; calls are asynchronous on
the current stream, or on `stream`: what they are given has to be ready there
and to live until it is done (Tensor.record_stream), and results that they
allocate belong to it.  One cache serves one stream at a time.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib
from .engine import Context, _device_view, _raw_stream, _results_on

_F32, _I32 = torch.float32, torch.int32
_F16_BITS = (torch.float16, torch.int16, torch.uint16)


class Kv4Cache:
    """KV cache of `streams` streams in 4 bits (qora_kv4_create)."""

    def __init__(self, ctx: Context, layers: int, num_heads: int, kv_heads: int, head_dim: int,
                 max_pos: int, streams: int, page_positions: int, pool_pages: int):
        self.ctx, self.layers, self.num_heads, self.kv_heads = ctx, layers, num_heads, kv_heads
        self.head_dim, self.max_pos, self.streams = head_dim, max_pos, streams
        self.page_positions, self.pool_pages = page_positions, pool_pages
        self.device, self._dev = f"cuda:{ctx.device}", ctx.device
        self._L = L = _lib.load()
        # a decode step makes a call per layer: the entry points are looked up once
        self._reserve, self._advance, self._append = L.qora_kv4_reserve, L.qora_kv4_advance, L.qora_kv4_append
        self._accept = L.qora_kv4_accept
        self._write, self._read, self._attend = L.qora_kv4_write, L.qora_kv4_read, L.qora_kv4_attend
        h = C.c_void_p()
        _lib.call("qora_kv4_create", ctx.h, layers, num_heads, kv_heads, head_dim, max_pos, streams,
                  page_positions, pool_pages, C.byref(h))
        self.h = h

    def __del__(self):
        if getattr(self, "h", None):
            self._L.qora_kv4_destroy(self.h)
            self.h = None

    def _typed(self, name: str, t: torch.Tensor, dtype, n: int, exact: bool = False) -> int:
        """Pointer of a contiguous tensor of the cache's device that holds at least (exact: just) n values of dtype."""
        if (t.dtype is not dtype or t.numel() < n or (exact and t.numel() != n) or t.get_device() != self._dev
                or not t.is_contiguous()):
            raise ValueError(f"{name}: expected {n} contiguous values of {dtype} on {self.device}, got {tuple(t.shape)} "
                             f"of {t.dtype} on {t.device}")
        return t.data_ptr()

    def _rows(self, name: str, t: torch.Tensor, n: int, width: int) -> int:
        """Pointer of n or more contiguous f32 rows of just `width` values (a wider row would be misread), or of the
        n * width values in one."""
        have = t.numel()
        if (t.dtype is not _F32 or not (have == n * width or (t.dim() and t.shape[0] > n and have == t.shape[0] * width))
                or t.get_device() != self._dev or not t.is_contiguous()):
            raise ValueError(f"{name}: expected {n} contiguous rows of {width} {_F32} on {self.device}, got "
                             f"{tuple(t.shape)} of {t.dtype} on {t.device}")
        return t.data_ptr()

    def _norm(self, name: str, t: torch.Tensor) -> int:
        if (t.dtype not in _F16_BITS or t.numel() != self.head_dim or t.get_device() != self._dev
                or not t.is_contiguous()):
            raise ValueError(f"{name}: expected {self.head_dim} f16 values (or their bits as int16) on {self.device}, "
                             f"got {tuple(t.shape)} of {t.dtype} on {t.device}")
        return t.data_ptr()

    def _stream(self, stream) -> int:
        return _raw_stream(self._dev) if stream is None else stream.cuda_stream

    def reset(self, ids=None, stream=None):
        """Empties the streams `ids` (all: None)."""
        if ids is None:
            _lib.call("qora_kv4_reset", self.h, None, 0, self._stream(stream))
        else:
            a = np.asarray(ids, np.int32)
            _lib.call("qora_kv4_reset", self.h, a.ctypes.data, a.size, self._stream(stream))

    def lengths(self, stream=None) -> np.ndarray:
        out = np.empty(self.streams, np.int32)
        _lib.call("qora_kv4_lengths_host", self.h, out.ctypes.data, self._stream(stream))
        return out

    def state(self) -> dict:
        """Views of the device state: table [streams][pages_per_stream] and
        lengths [streams], int32.  A view keeps the cache alive."""
        table, per, lengths = C.c_void_p(), C.c_int32(), C.c_void_p()
        _lib.call("qora_kv4_state", self.h, C.byref(table), C.byref(per), C.byref(lengths))
        return {"table": _device_view(table.value, (self.streams, per.value), "<i4", self.device, self),
                "lengths": _device_view(lengths.value, (self.streams,), "<i4", self.device, self)}

    def reserve(self, counts: torch.Tensor, max_tokens: int, out=None, stream=None):
        """Maps pages for counts[b] new tokens per stream (int32 [streams]);
        returns (slots [max_tokens], positions [max_tokens], offsets [streams + 1])."""
        if out is None:
            i32 = dict(dtype=torch.int32, device=self.device)
            with _results_on(stream):
                out = (torch.empty(max_tokens, **i32), torch.empty(max_tokens, **i32),
                       torch.empty(self.streams + 1, **i32))
        slots, positions, offsets = out
        rc = self._reserve(self.h, self._typed("counts", counts, _I32, self.streams, True), max_tokens,
                           self._typed("slots", slots, _I32, max_tokens),
                           self._typed("positions", positions, _I32, max_tokens),
                           self._typed("offsets", offsets, _I32, self.streams + 1, True), self._stream(stream))
        if rc:
            _lib.check(rc, "qora_kv4_reserve")
        return out

    def advance(self, counts: torch.Tensor, stream=None, offsets: torch.Tensor | None = None):
        """Adds counts[b] (int32 [streams]; negative: rolls back) to the lengths.
        With `offsets` from `reserve`, a stream moves by at most the tokens that
        were reserved for it: none without tokens, none after a refusal."""
        n = self._typed("counts", counts, _I32, self.streams, True)
        if offsets is None:
            rc = self._advance(self.h, n, self._stream(stream))
        else:
            rc = self._accept(self.h, n, self._typed("offsets", offsets, _I32, self.streams + 1, True), self._stream(stream))
        if rc:
            _lib.check(rc, "qora_kv4_advance")

    def append(self, layer: int, qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
               rope_cos: torch.Tensor, rope_sin: torch.Tensor, positions: torch.Tensor,
               slots: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """qk-norm, RoPE and 4-bit append of one layer: qkv [n][q|k|v] raw
        projections; q_norm / k_norm f16 (or its bits as int16); returns the
        normed and rotated queries [n][num_heads * head_dim]."""
        n, hd = qkv.shape[0], self.head_dim
        if out is None:
            with _results_on(stream):
                out = torch.empty(n, self.num_heads * hd, device=qkv.device)
        table, half = rope_cos.numel(), hd // 2
        if table % half or (rope_cos.dim() > 1 and rope_cos.shape[-1] != half):
            raise ValueError(f"rope_cos: expected rows of {half} angles, got {tuple(rope_cos.shape)}")
        rc = self._append(self.h, layer, self._rows("qkv", qkv, n, (self.num_heads + 2 * self.kv_heads) * hd),
                          self._norm("q_norm", q_norm), self._norm("k_norm", k_norm),
                          self._typed("rope_cos", rope_cos, _F32, 0), self._typed("rope_sin", rope_sin, _F32, table, True),
                          table // half, self._typed("positions", positions, _I32, n),
                          self._typed("slots", slots, _I32, n), n,
                          self._rows("out", out, n, self.num_heads * hd), self._stream(stream))
        if rc:
            _lib.check(rc, "qora_kv4_append")
        return out

    def write(self, layer: int, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, stream=None):
        """Stores rows of keys (normed, rotated) and values [n][kv_heads * head_dim]."""
        n = slots.numel()
        width = self.kv_heads * self.head_dim
        rc = self._write(self.h, layer, self._typed("slots", slots, _I32, n), n, self._rows("k", k, n, width),
                         self._rows("v", v, n, width), self._stream(stream))
        if rc:
            _lib.check(rc, "qora_kv4_write")

    def read(self, layer: int, slots: torch.Tensor, out=None, stream=None):
        """The keys and values that the slots hold, f32 [n][kv_heads * head_dim]
        (rows of slot -1 are left as they were)."""
        n = slots.numel()
        width = self.kv_heads * self.head_dim
        if out is None:
            with _results_on(stream):
                out = tuple(torch.zeros(n, width, device=slots.device) for _ in range(2))
        k, v = out
        rc = self._read(self.h, layer, self._typed("slots", slots, _I32, n), n, self._rows("k", k, n, width),
                        self._rows("v", v, n, width), self._stream(stream))
        if rc:
            _lib.check(rc, "qora_kv4_read")
        return out

    def attend(self, layer: int, q: torch.Tensor, offsets: torch.Tensor, max_count: int,
               out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """Attention of one layer for the tokens that `offsets` lists: q
        [n][num_heads * head_dim] from `append`; max_count bounds the tokens of
        one stream (1 in a decode step).  Returns [n][num_heads * head_dim]."""
        n, width = q.shape[0], self.num_heads * self.head_dim
        if out is None:
            with _results_on(stream):
                out = torch.empty(n, width, device=q.device)
        rc = self._attend(self.h, layer, self._rows("q", q, n, width),
                          self._typed("offsets", offsets, _I32, self.streams + 1, True), n, max_count,
                          self._rows("out", out, n, width), self._stream(stream))
        if rc:
            _lib.check(rc, "qora_kv4_attend")
        return out
