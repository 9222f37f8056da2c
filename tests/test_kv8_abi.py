"""CPU: what the 8-bit K/V cache's entry points refuse (``animaxs_kv8_*``), without a GPU, and the CPU oracle's own
rounding."""
import ctypes

import numpy as np
import pytest

from oracle import kv8_oracle as ora


@pytest.fixture(scope="module")
def lib():
    from animaxs_b200 import _lib
    return _lib.lib()


def _cache(**kw):
    from animaxs_b200._lib import Kv8Cache
    c = Kv8Cache(2, 512, 8, 128, 0, 0x1000, 0x2000, 0x3000, 0x4000)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _write(lib, cache=None, k=0x5000, v=0x6000, **kw):
    from animaxs_b200._lib import Kv8WriteDesc
    d = Kv8WriteDesc(16, 0, None, None, 1024, 128, 16384, 1024, 128, 16384)
    for name, x in kw.items():
        setattr(d, name, x)
    c = _cache() if cache is None else cache
    return lib.animaxs_kv8_write_validate(None, ctypes.byref(c), ctypes.byref(d), k, v)


def _attn(lib, cache=None, q=0x5000, o=0x6000, q_len=3, kv_len=512, heads=16, **kw):
    from animaxs_b200._lib import AttnDesc
    d = AttnDesc()
    lib.animaxs_attn_desc_init(ctypes.byref(d), 2, heads, 8, q_len, kv_len, 128)
    for name, x in kw.items():
        setattr(d, name, x)
    c = _cache() if cache is None else cache
    return lib.animaxs_kv8_attn_validate(None, ctypes.byref(c), ctypes.byref(d), q, o)


def test_cache_bytes(lib):
    a, b = ctypes.c_int64(), ctypes.c_int64()
    assert lib.animaxs_kv8_cache_bytes(2, 130, 8, 128, ctypes.byref(a), ctypes.byref(b)) == 0
    assert (a.value, b.value) == (2 * 130 * 8 * 128, 2 * 8 * 3 * 4)
    assert lib.animaxs_kv8_cache_bytes(2, 130, 8, 96, ctypes.byref(a), ctypes.byref(b)) == -2
    assert lib.animaxs_kv8_cache_bytes(2, 0, 8, 64, ctypes.byref(a), ctypes.byref(b)) == -1
    assert lib.animaxs_kv8_cache_bytes(1 << 20, 1 << 30, 64, 128, ctypes.byref(a), ctypes.byref(b)) == -8


@pytest.mark.parametrize("bad,code", [
    ({"batch": 0}, -1), ({"capacity": -3}, -1), ({"kv_heads": 0}, -1), ({"head_dim": 256}, -2), ({"format": 2}, -1),
    ({"k_codes": None}, -1), ({"v_scale": None}, -1), ({"v_codes": 0x2008}, -1), ({"k_scale": 0x3002}, -1),
    ({"batch": 1 << 20, "kv_heads": 1 << 12}, -8)])
def test_cache_refusals(lib, bad, code):
    assert _write(lib, _cache(**bad)) == code
    assert _attn(lib, _cache(**bad)) == code


def test_write_refusals(lib):
    assert _write(lib) == 0
    assert _write(lib, k=None) == -1
    assert _write(lib, v=0x6008) == -1
    assert _write(lib, tokens=0) == -1
    assert _write(lib, start=-1) == -3
    assert _write(lib, start=496) == 0
    assert _write(lib, start=497) == -3
    assert _write(lib, start=497, starts=0x7000) == 0       # per-sequence positions are checked on the device
    assert _write(lib, k_tok_stride=1020) == -1
    assert _write(lib, v_head_stride=-128) == -1
    assert _write(lib, k_tok_stride=0) == -1
    assert _write(lib, v_head_stride=0) == -1
    assert _write(lib, k_batch_stride=0) == 0               # one source for every sequence
    assert _write(lib, v_batch_stride=1 << 40) == -8
    assert lib.animaxs_kv8_write(None, None, None, None, None, None) == -1
    assert lib.animaxs_kv8_read(None, None, 0, 1, None, None, None, 0, 0, 0, None) == -1


def test_attention_refusals(lib):
    assert _attn(lib) == 0
    assert _attn(lib, causal=1) == 0                        # q_len and kv_len are independent
    assert _attn(lib, kv_len=513) == -3
    assert _attn(lib, kv_len=0) == -1
    assert _attn(lib, q_len=0) == -1
    assert _attn(lib, heads=12) == -1
    assert _attn(lib, batch=1) == -1
    assert _attn(lib, head_dim=64) == -1
    assert _attn(lib, q=None) == -1
    assert _attn(lib, o=0x6004) == -1
    assert _attn(lib, q_tok_stride=2047) == -1
    assert _attn(lib, o_batch_stride=0) == -1
    assert _attn(lib, q_batch_stride=0) == 0
    assert _attn(lib, o_bytes=8) == -3
    assert _attn(lib, qk_norm=1) == -2                      # K is normalised before it is written
    assert _attn(lib, qk_norm=1, qk_norm_targets=1) == 0
    assert _attn(lib, qk_norm=2, qk_norm_targets=1) == -2
    assert _attn(lib, numerics=1) == -2
    assert _attn(lib, numerics=2) == -2
    assert _attn(lib, scale=float("nan")) == -1
    assert _attn(lib, kv_valid_len=513) == -1
    assert lib.animaxs_kv8_attn_forward(None, None, None, None, None, None) == -1


def test_oracle_e4m3_rounding_against_torch():
    import torch
    x = np.concatenate([np.linspace(-460, 460, 20001), np.geomspace(1e-4, 1, 5001)]).astype(np.float32)
    want = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ora.round_e4m3(x), want)
