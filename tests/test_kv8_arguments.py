"""CPU: what ``QuantizedKVCache`` refuses before a pointer reaches the device, with stand-ins for device tensors and
for the library."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from animaxs_b200 import AttentionValidationError, QuantizedKVCache, _lib


class Tensor:
    """A device tensor as far as the cache looks at one."""

    def __init__(self, *shape, dtype=torch.float16, device=0, stride=None):
        self.shape, self.dtype, self._device = torch.Size(shape), dtype, device
        self._stride = torch.empty(shape, device="meta").stride() if stride is None else stride
        self.is_cuda = device >= 0
        self.device = SimpleNamespace(type="cuda" if device >= 0 else "cpu", index=device if device >= 0 else None)

    def get_device(self):
        return self._device

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i=None):
        return self._stride if i is None else self._stride[i]

    def is_contiguous(self):
        return self._stride == torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        return 0x10000


class Library:
    """Accepts every call and keeps the last one's arguments."""

    def __init__(self):
        self.calls = []

    def animaxs_attn_desc_init(self, *args):
        return _lib.lib().animaxs_attn_desc_init(*args)

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture()
def cache():
    """A cache of 2 sequences, 100 positions, 4 heads of 64 on device 0."""
    from animaxs_b200 import AttentionExecutor
    lib = Library()
    ex = AttentionExecutor.__new__(AttentionExecutor)
    ex.device, ex.numerics, ex.layout, ex._lib, ex._ctx = 0, "legacy", None, lib, ctypes.c_void_p(1)
    ex.close = lambda: None
    c = QuantizedKVCache.__new__(QuantizedKVCache)
    codes, scale = Tensor(2, 4, 100, 64, dtype=torch.int8), Tensor(2, 4, 2, dtype=torch.float32)
    c._bind(ex, codes, codes, scale, scale)
    c._stream = lambda stream: 0
    c.lib = lib
    yield c
    ex._ctx = None


def _calls(cache, **kw):
    """The three calls, with some arguments replaced."""
    h = kw.get("h", Tensor(2, 10, 4, 64))
    ints = kw.get("ints")
    return {
        "write k": lambda: cache.write(h, Tensor(2, 10, 4, 64), starts=ints),
        "write v": lambda: cache.write(Tensor(2, 10, 4, 64), h, counts=ints),
        "read k": lambda: cache.read(0, 10, k_out=h, v_out=Tensor(2, 10, 4, 64), lens=ints),
        "read v": lambda: cache.read(0, 10, k_out=Tensor(2, 10, 4, 64), v_out=h, lens=ints),
        "attend q": lambda: cache.attention(h, Tensor(2, 10, 4, 64), lens=ints),
        "attend out": lambda: cache.attention(Tensor(2, 10, 4, 64), h, lens=ints),
    }


def _refused(cache, call):
    before = len(cache.lib.calls)
    with pytest.raises(AttentionValidationError):
        call()
    assert len(cache.lib.calls) == before


def test_good_calls_reach_the_library(cache):
    for call in _calls(cache, ints=Tensor(2, dtype=torch.int32)).values():
        before = len(cache.lib.calls)
        call()
        assert len(cache.lib.calls) == before + 1


@pytest.mark.parametrize("weight", [
    Tensor(64, dtype=torch.float32), Tensor(64, dtype=torch.bfloat16), Tensor(32), Tensor(128), Tensor(64, device=-1),
    Tensor(64, stride=(2,))], ids=["fp32", "bf16", "short", "long", "host", "strided"])
def test_norm_weight(cache, weight):
    q, out = Tensor(2, 10, 4, 64), Tensor(2, 10, 4, 64)
    cache.attention(q, out, qk_norm="rms", q_norm_weight=Tensor(64))
    _refused(cache, lambda: cache.attention(q, out, qk_norm="rms", q_norm_weight=weight))


@pytest.mark.parametrize("device", [-1, 1])
@pytest.mark.parametrize("call", ["write k", "write v", "read k", "read v", "attend q", "attend out"])
def test_tensors_of_another_device(cache, device, call):
    """The host's, or another GPU's; also where a tensor of the same shape went through before."""
    for _ in range(2):
        _refused(cache, _calls(cache, h=Tensor(2, 10, 4, 64, device=device))[call])
        _refused(cache, _calls(cache, ints=Tensor(2, dtype=torch.int32, device=device))[call])
        _calls(cache)[call]()
    _refused(cache, lambda: cache.attention(Tensor(2, 10, 4, 64), Tensor(2, 10, 4, 64), qk_norm="rms",
                                            q_norm_weight=Tensor(64, device=device)))


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 5, -(1 << 32) + 5, 1 << 64])
def test_integers_past_32_bits(cache, n):
    """Not cut to their low bits, which name other positions."""
    h, out = Tensor(2, 10, 4, 64), Tensor(2, 10, 4, 64)
    for call in (lambda: cache.write(h, h, n), lambda: cache.read(n, 10, k_out=h, v_out=out),
                 lambda: cache.read(5, n, k_out=h, v_out=out), lambda: cache.read(n, k_out=h, v_out=out),
                 lambda: cache.attention(h, out, kv_len=n)):
        _refused(cache, call)
    if n > 0:
        wide = Tensor(2, n, 4, 64, stride=(0, 8, 64, 1)) if n < 1 << 60 else h
        if wide is not h:
            _refused(cache, lambda: cache.write(wide, wide))
            _refused(cache, lambda: cache.attention(wide, wide))
    lib = cache.lib
    for what in ("batch", "capacity", "kv_heads", "head_dim"):
        before = len(lib.calls)
        with pytest.raises(AttentionValidationError):
            QuantizedKVCache(cache.ex, **{what: n})
        assert len(lib.calls) == before


@pytest.mark.parametrize("start,tokens", [(95, 10), (101, None), (-1, 5), (-5, None), (0, -1), (3, 98)])
def test_read_outside_the_capacity(cache, start, tokens):
    """Refused as every other bad argument is, before outputs are made."""
    _refused(cache, lambda: cache.read(start, tokens))
