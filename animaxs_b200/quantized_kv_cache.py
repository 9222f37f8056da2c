"""An 8-bit K/V cache (``animaxs_kv8_*`` in ``include/animaxs_attn.h``).

Half the memory of an fp16 cache and half the bytes attention reads: ``[batch][kv_heads][capacity][head_dim]``
codes, int8 or e4m3, for K and for V, with one fp32 scale for each head and block of 64 tokens.  The reference
has no counterpart (its caches are fp16, AnimaXS/Runtime/Metal/DiTBlockExecutor.swift:19-43).  It serves the
same cross-attention K/V of a block, written once per generation (:1105-1161), and sequences that grow token
by token, which the reference does not have (its text encoder runs each prompt in one causal call).  The caller
keeps each sequence's length.
"""

from __future__ import annotations

import ctypes

from . import _lib
from ._lib import AttentionValidationError, Kv8Cache, Kv8WriteDesc, raise_for
from .executor import AttentionExecutor, AttentionInputLayout

_FORMATS = {"int8": _lib.KV8_INT8, "e4m3": _lib.KV8_E4M3}


def _current_stream(device):
    """The current stream's handle.  The first call finds out how to get it without a Stream object (0.1 us of a call
    that takes 8 in all, not 1.3), so that importing the package does not import torch."""
    global _current_stream
    try:
        from torch._C import _cuda_getCurrentRawStream as get
    except ImportError:
        import torch

        def get(device):
            return torch.cuda.current_stream(device).cuda_stream
    _current_stream = get
    return get(device)


def _invalid(message):
    return AttentionValidationError(_lib.ERR_INVALID_ARG, message)


def _int32(value, what):
    """``value`` as the C ABI's 32-bit integer; ctypes would drop the bits above without a word."""
    value = int(value)
    if not -0x80000000 <= value <= 0x7fffffff:
        raise AttentionValidationError(_lib.ERR_OVERFLOW, f"{what} {value} does not fit 32 bits")
    return value


class QuantizedKVCache:
    """One layer's K and V of ``batch`` sequences on the executor's device.

    ``k_codes`` / ``v_codes`` are ``[batch, kv_heads, capacity, head_dim]`` (``torch.int8`` or
    ``torch.float8_e4m3fn``), ``k_scale`` / ``v_scale`` fp32 ``[batch, kv_heads, ceil(capacity / 64)]``.
    Work is enqueued on ``stream`` (default: the current torch stream)."""

    block_tokens = _lib.KV8_BLOCK_TOKENS

    def __init__(self, executor: AttentionExecutor, batch: int = 1, capacity: int = 512, kv_heads: int = 16,
                 head_dim: int = 128, format: str = "int8"):
        import torch
        if format not in _FORMATS:
            raise _invalid(f"unknown 8-bit K/V cache format {format!r}")
        code_bytes, scale_bytes = ctypes.c_int64(), ctypes.c_int64()
        for what, x in (("batch", batch), ("capacity", capacity), ("kv_heads", kv_heads), ("head_dim", head_dim)):
            _int32(x, what)
        rc = executor._lib.animaxs_kv8_cache_bytes(batch, capacity, kv_heads, head_dim, ctypes.byref(code_bytes),
                                                   ctypes.byref(scale_bytes))
        raise_for(rc, "invalid 8-bit K/V cache shape (head_dim 64 or 128, positive sizes)")
        dev = torch.device("cuda", executor.device)
        dtype = torch.int8 if format == "int8" else torch.float8_e4m3fn
        # Zeros: a key that a causal mask hides still meets a weight of 0, which a NaN code (e4m3 has them) would turn
        # into NaN where ``lens`` counts positions not written yet, as a padded batch of prompts does; and a write
        # that starts inside a block nothing was written to finds no scale there.
        codes = [torch.zeros((batch, kv_heads, capacity, head_dim), dtype=torch.int8, device=dev).view(dtype)
                 for _ in range(2)]
        blocks = scale_bytes.value // 4 // (batch * kv_heads)
        scales = [torch.zeros((batch, kv_heads, blocks), dtype=torch.float32, device=dev) for _ in range(2)]
        self._bind(executor, *codes, *scales)

    @classmethod
    def wrap(cls, executor: AttentionExecutor, k_codes, v_codes, k_scale, v_scale) -> "QuantizedKVCache":
        """A cache over existing (contiguous) tensors, for example one layer of a larger allocation."""
        self = cls.__new__(cls)
        self._bind(executor, k_codes, v_codes, k_scale, v_scale)
        return self

    def _bind(self, executor, k_codes, v_codes, k_scale, v_scale):
        import torch
        formats = {torch.int8: "int8", torch.float8_e4m3fn: "e4m3"}
        if k_codes.dtype not in formats or v_codes.dtype != k_codes.dtype:
            raise _invalid("codes must be torch.int8 or torch.float8_e4m3fn")
        if k_codes.dim() != 4 or v_codes.shape != k_codes.shape:
            raise _invalid("codes must be [batch, kv_heads, capacity, head_dim]")
        b, h, cap, d = k_codes.shape
        blocks = (b, h, -(-cap // self.block_tokens))
        for t in (k_scale, v_scale):
            if t.dtype != torch.float32 or tuple(t.shape) != blocks:
                raise _invalid(f"scales must be float32 {list(blocks)}")
        for t in (k_codes, v_codes, k_scale, v_scale):
            if not t.is_contiguous() or not t.is_cuda or t.device.index != executor.device:
                raise _invalid("cache tensors must be contiguous, on the executor's device")
        self.ex = executor
        self._lib = executor._lib
        self.format = formats[k_codes.dtype]
        self.batch, self.kv_heads, self.capacity, self.head_dim = b, h, cap, d
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self._c = Kv8Cache(b, cap, h, d, _FORMATS[self.format], k_codes.data_ptr(), v_codes.data_ptr(),
                           k_scale.data_ptr(), v_scale.data_ptr())
        self._cref = ctypes.byref(self._c)
        self._descs = {}

    @property
    def nbytes(self) -> int:
        """Bytes of the codes and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale))

    def _stream(self, stream):
        if stream is None:
            return _current_stream(self.ex.device)
        return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)

    def _ints(self, t, what):
        """Device pointer of a per-sequence int32 tensor (0 for None)."""
        if t is None:
            return None
        import torch
        if t.dtype != torch.int32 or t.numel() != self.batch or t.get_device() != self.ex.device \
                or not t.is_contiguous():
            raise _invalid(f"{what} must be a contiguous int32 tensor of {self.batch} values on the executor's device")
        return t.data_ptr()

    def _view(self, t, tokens, heads, what):
        import torch
        if t.dtype != torch.float16 or t.get_device() != self.ex.device or t.dim() != 4 or t.shape[0] != self.batch \
                or t.shape[2] != heads or t.shape[3] != self.head_dim or (tokens is not None and t.shape[1] != tokens):
            raise _invalid(f"{what} must be fp16 [{self.batch}, tokens, {heads}, {self.head_dim}] on the "
                           "executor's device")
        if t.stride(3) != 1:
            raise _invalid("head_dim must be contiguous")
        _int32(t.shape[1], "token count")

    def write(self, k, v, start: int = 0, *, starts=None, counts=None, stream=None) -> None:
        """Quantise ``k`` and ``v`` (``[batch, tokens, kv_heads, head_dim]`` fp16, any strides) into positions
        ``start + t`` (``starts``: int32 device tensor, one per sequence; ``counts``: only the first ``counts[b]``
        tokens).  Appending to a half-filled block keeps its older tokens, re-rounded where the block's scale
        grows.  Positions that ``starts`` puts outside the capacity are not written."""
        import torch
        key = ("w", k.shape, v.shape, k.stride(), v.stride())
        d = self._descs.get(key)
        if d is None:
            self._view(k, None, self.kv_heads, "k")
            self._view(v, k.shape[1], self.kv_heads, "v")
            if k.shape[1] == 0:
                return
            d = Kv8WriteDesc(k.shape[1], 0, None, None, k.stride(1), k.stride(2), k.stride(0), v.stride(1),
                             v.stride(2), v.stride(0))
            self._remember(key, d)
        dev = self.ex.device
        if k.dtype != torch.float16 or v.dtype != torch.float16 or k.get_device() != dev or v.get_device() != dev:
            raise _invalid("k and v must be fp16 on the executor's device")
        d.start = _int32(start, "position")
        d.starts = self._ints(starts, "starts")
        d.counts = self._ints(counts, "counts")
        rc = self._lib.animaxs_kv8_write(self.ex._ctx, self._cref, ctypes.byref(d), k.data_ptr(), v.data_ptr(),
                                         self._stream(stream))
        if rc:
            self.ex._check(rc)

    def read(self, start: int = 0, tokens: int | None = None, *, lens=None, k_out=None, v_out=None, stream=None):
        """Positions ``[start, start + tokens)`` as fp16 ``(k, v)``, each ``[batch, tokens, kv_heads, head_dim]``;
        rows at or past position ``lens[b]`` are zeros."""
        import torch
        start = _int32(start, "position")
        tokens = self.capacity - start if tokens is None else _int32(tokens, "token count")
        if tokens < 0 or (tokens > 0 and (start < 0 or start + tokens > self.capacity)):
            raise AttentionValidationError(
                _lib.ERR_OOB, f"positions [{start}, {start + tokens}) outside the cache's capacity {self.capacity}")
        if k_out is None or v_out is None:
            like = self._descs.get(("r", tokens))  # of the outputs' shape, without memory of its own
            if like is None:
                like = self.k_scale.new_empty((), dtype=torch.float16).expand(self.batch, tokens, self.kv_heads,
                                                                              self.head_dim)
                self._remember(("r", tokens), like)
        if k_out is None:
            k_out = torch.empty_like(like, memory_format=torch.contiguous_format)
        else:
            self._view(k_out, tokens, self.kv_heads, "k_out")
        if v_out is None:
            v_out = torch.empty_like(like, memory_format=torch.contiguous_format)
        else:
            self._view(v_out, tokens, self.kv_heads, "v_out")
        if k_out.stride() != v_out.stride():
            raise _invalid("k_out and v_out must have the same strides")
        if tokens == 0:
            return k_out, v_out
        sb, st, sh, _ = k_out.stride()
        rc = self._lib.animaxs_kv8_read(self.ex._ctx, self._cref, start, tokens, self._ints(lens, "lens"),
                                        k_out.data_ptr(), v_out.data_ptr(), st, sh, sb, self._stream(stream))
        if rc:
            self.ex._check(rc)
        return k_out, v_out

    def attention(self, q, out=None, *, lens=None, kv_len: int | None = None, causal: bool = False, scale=None,
                  qk_norm: str = "none", q_norm_weight=None, eps: float = 1e-6, stream=None):
        """``softmax(scale * q k^T + mask) v`` over the cache for ``q`` ``[batch, q_len, heads, head_dim]`` fp16, any
        strides.  ``kv_len`` (default: the capacity) is the most tokens any sequence has, ``lens`` (int32 device
        tensor) each one's own length.  ``causal``: the queries are the last ``q_len`` tokens of their sequence.  A
        query that sees no key gets zeros.  ``qk_norm="rms"`` normalises q first (K is normalised before it is written)."""
        import torch
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)  # 1 us less than new_empty
            key = ("a", q.shape, q.stride(), kv_len, causal, scale, qk_norm, eps)
        else:
            key = ("o", q.shape, q.stride(), kv_len, causal, scale, qk_norm, eps, out.shape, out.stride())
        d = self._descs.get(key)
        if d is None:
            self._view(q, None, q.shape[2] if q.dim() == 4 else 0, "q")
            self._view(out, q.shape[1], q.shape[2], "out")
            if q.shape[1] == 0:
                return out
            d = self.ex.make_desc(heads=q.shape[2], query_count=q.shape[1],
                                  key_count=self.capacity if kv_len is None else _int32(kv_len, "kv_len"),
                                  head_dim=self.head_dim, key_value_heads=self.kv_heads, causal=causal,
                                  layout=AttentionInputLayout.head_major, qk_norm=qk_norm, qk_norm_targets="q",
                                  eps=eps, scale=scale, batch=self.batch)
            d.q_batch_stride, d.q_tok_stride, d.q_head_stride, _ = q.stride()
            d.o_batch_stride, d.o_tok_stride, d.o_head_stride, _ = out.stride()
            self._remember(key, d)
        dev = self.ex.device
        if q.dtype != torch.float16 or out.dtype != torch.float16 or q.get_device() != dev or out.get_device() != dev:
            raise _invalid("q and out must be fp16 on the executor's device")
        d.kv_valid_lens = self._ints(lens, "lens")
        if q_norm_weight is not None and (
                q_norm_weight.dtype != torch.float16 or q_norm_weight.numel() != self.head_dim
                or q_norm_weight.get_device() != dev or not q_norm_weight.is_contiguous()):
            raise _invalid(f"q_norm_weight must be a contiguous fp16 tensor of {self.head_dim} values on the "
                           "executor's device")
        d.q_norm_weight = None if q_norm_weight is None else q_norm_weight.data_ptr()
        rc = self._lib.animaxs_kv8_attn_forward(self.ex._ctx, self._cref, ctypes.byref(d), q.data_ptr(),
                                                out.data_ptr(), self._stream(stream))
        if rc:
            self.ex._check(rc)
        return out

    def _remember(self, key, desc):
        if len(self._descs) > 256:
            self._descs.clear()
        self._descs[key] = desc
