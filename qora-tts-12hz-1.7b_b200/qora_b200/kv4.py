"""The 4-bit paged KV cache (qora_kv4): block tables built on the GPU, the
append with qk-norm and rotation, and attention over the cache.

A speculative decode step of every stream, without a return to the host:

    slots, positions, offsets = kv.reserve(counts, max_tokens)
    for each layer:
        q = kv.append(layer, qkv, q_norm, k_norm, cos, sin, positions, slots)
        o = kv.attend(layer, q, offsets, max_count)
    tokens, n_out = engine.verify_drafts(ctx, drafts, draft_probs, target_probs, uniforms)
    kv.advance(n_out)

Tensors are on the context's device and contiguous; calls are asynchronous on
the current stream (or `stream`).  One cache serves one stream at a time.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib
from .engine import Context, _device_view, _dp




class Kv4Cache:
    """KV cache of `streams` streams in 4 bits (qora_kv4_create)."""

    def __init__(self, ctx: Context, layers: int, num_heads: int, kv_heads: int, head_dim: int,
                 max_pos: int, streams: int, page_positions: int, pool_pages: int):
        self.ctx, self.layers, self.num_heads, self.kv_heads = ctx, layers, num_heads, kv_heads
        self.head_dim, self.max_pos, self.streams = head_dim, max_pos, streams
        self.page_positions, self.pool_pages = page_positions, pool_pages
        self.device = f"cuda:{ctx.device}"
        self._L = _lib.load()
        h = C.c_void_p()
        _lib.call("qora_kv4_create", ctx.h, layers, num_heads, kv_heads, head_dim, max_pos, streams,
                  page_positions, pool_pages, C.byref(h))
        self.h = h

    def __del__(self):
        if getattr(self, "h", None):
            self._L.qora_kv4_destroy(self.h)
            self.h = None

    def _typed(self, name: str, t: torch.Tensor, dtype, n: int) -> int:
        """Pointer of a tensor of the cache's device that must hold at least n values of dtype."""
        if t.dtype != dtype or t.numel() < n or not t.is_cuda or t.device.index != self.ctx.device:
            raise ValueError(f"{name}: expected {n} values of {dtype} on {self.device}, got {tuple(t.shape)} of "
                             f"{t.dtype} on {t.device}")
        return _dp(t)

    def _stream(self, stream) -> int:
        return (stream if stream is not None else torch.cuda.current_stream(self.ctx.device)).cuda_stream

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
            out = (torch.empty(max_tokens, **i32), torch.empty(max_tokens, **i32),
                   torch.empty(self.streams + 1, **i32))
        slots, positions, offsets = out
        _lib.call("qora_kv4_reserve", self.h, self._typed("counts", counts, torch.int32, self.streams), max_tokens,
                  self._typed("slots", slots, torch.int32, max_tokens),
                  self._typed("positions", positions, torch.int32, max_tokens),
                  self._typed("offsets", offsets, torch.int32, self.streams + 1), self._stream(stream))
        return out

    def advance(self, counts: torch.Tensor, stream=None):
        """Adds counts[b] (int32 [streams]; negative: rolls back) to the lengths."""
        _lib.call("qora_kv4_advance", self.h, self._typed("counts", counts, torch.int32, self.streams),
                  self._stream(stream))

    def append(self, layer: int, qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
               rope_cos: torch.Tensor, rope_sin: torch.Tensor, positions: torch.Tensor,
               slots: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """qk-norm, RoPE and 4-bit append of one layer: qkv [n][q|k|v] raw
        projections; q_norm / k_norm f16 (or its bits as int16); returns the
        normed and rotated queries [n][num_heads * head_dim]."""
        n, width = qkv.shape[0], (self.num_heads + 2 * self.kv_heads) * self.head_dim
        if out is None:
            out = torch.empty(n, self.num_heads * self.head_dim, device=qkv.device)
        if q_norm.element_size() != 2 or k_norm.element_size() != 2 or min(q_norm.numel(), k_norm.numel()) < self.head_dim:
            raise ValueError(f"q_norm / k_norm: expected {self.head_dim} f16 values")
        rope_max = rope_cos.numel() // (self.head_dim // 2)
        _lib.call("qora_kv4_append", self.h, layer, self._typed("qkv", qkv, torch.float32, n * width), _dp(q_norm),
                  _dp(k_norm), self._typed("rope_cos", rope_cos, torch.float32, 0),
                  self._typed("rope_sin", rope_sin, torch.float32, rope_cos.numel()), rope_max,
                  self._typed("positions", positions, torch.int32, n), self._typed("slots", slots, torch.int32, n), n,
                  self._typed("out", out, torch.float32, n * self.num_heads * self.head_dim), self._stream(stream))
        return out

    def write(self, layer: int, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, stream=None):
        """Stores rows of keys (normed, rotated) and values [n][kv_heads * head_dim]."""
        n = slots.numel()
        want = n * self.kv_heads * self.head_dim
        _lib.call("qora_kv4_write", self.h, layer, self._typed("slots", slots, torch.int32, n), n,
                  self._typed("k", k, torch.float32, want), self._typed("v", v, torch.float32, want), self._stream(stream))

    def read(self, layer: int, slots: torch.Tensor, out=None, stream=None):
        """The keys and values that the slots hold, f32 [n][kv_heads * head_dim]
        (rows of slot -1 are left as they were)."""
        n = slots.numel()
        want = n * self.kv_heads * self.head_dim
        if out is None:
            out = tuple(torch.zeros(n, self.kv_heads * self.head_dim, device=slots.device) for _ in range(2))
        k, v = out
        _lib.call("qora_kv4_read", self.h, layer, self._typed("slots", slots, torch.int32, n), n,
                  self._typed("k", k, torch.float32, want), self._typed("v", v, torch.float32, want), self._stream(stream))
        return out

    def attend(self, layer: int, q: torch.Tensor, offsets: torch.Tensor, max_count: int,
               out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """Attention of one layer for the tokens that `offsets` lists: q
        [n][num_heads * head_dim] from `append`; max_count bounds the tokens of
        one stream (1 in a decode step).  Returns [n][num_heads * head_dim]."""
        n, width = q.shape[0], self.num_heads * self.head_dim
        if out is None:
            out = torch.empty(n, width, device=q.device)
        _lib.call("qora_kv4_attend", self.h, layer, self._typed("q", q, torch.float32, n * width),
                  self._typed("offsets", offsets, torch.int32, self.streams + 1), n, max_count,
                  self._typed("out", out, torch.float32, n * width), self._stream(stream))
        return out
