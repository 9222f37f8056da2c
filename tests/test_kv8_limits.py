"""CPU: sizes at which the 8-bit K/V cache's launches reach 32 bits are refused, not cut."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from animaxs_b200 import _lib
    return _lib.lib()


def _write(lib, batch, capacity, kv_heads, tokens):
    from animaxs_b200._lib import Kv8Cache, Kv8WriteDesc
    c = Kv8Cache(batch, capacity, kv_heads, 64, 0, 0x1000, 0x2000, 0x3000, 0x4000)
    d = Kv8WriteDesc(tokens, 0, 0x7000, None, 64 * kv_heads, 64, 1 << 20, 64 * kv_heads, 64, 1 << 20)
    return lib.animaxs_kv8_write_validate(None, ctypes.byref(c), ctypes.byref(d), 0x5000, 0x6000)


@pytest.mark.parametrize("batch,capacity,kv_heads,tokens,code", [
    (2, 512, 8, (1 << 31) - 1, 0),           # positions past the capacity are not written: 8 blocks a head
    (2, 512, 8, (1 << 31) - 62, 0),
    (64, 1 << 30, 8, (1 << 31) - 1, -8),     # 2 x 512 heads x 2^24 blocks
    (64, 1 << 30, 1, (1 << 31) - 1, -8),
    (63, 1 << 30, 1, (1 << 31) - 1, 0),
    (64, 1 << 30, 8, 1 << 20, 0), (1 << 30, 1, 1, 1, -8), ((1 << 30) - 1, 1, 1, 1, 0)])
def test_blocks_of_a_write(lib, batch, capacity, kv_heads, tokens, code):
    assert _write(lib, batch, capacity, kv_heads, tokens) == code


@pytest.mark.parametrize("heads,q_len,code", [
    (1, (1 << 31) - 257, 0), (1, (1 << 31) - 256, -8), (1, (1 << 31) - 1, -8), (16, (1 << 27) - 17, 0),
    (16, (1 << 27) - 1, -8), (4, 1 << 29, -8)])
def test_query_rows(lib, heads, q_len, code):
    """Rows are numbered in 32 bits up to the end of the last pair of 128-row tiles."""
    from animaxs_b200._lib import AttnDesc, Kv8Cache
    c = Kv8Cache(1, 512, 1, 64, 0, 0x1000, 0x2000, 0x3000, 0x4000)
    d = AttnDesc()
    lib.animaxs_attn_desc_init(ctypes.byref(d), 1, heads, 1, q_len, 512, 64)
    d.q_tok_stride = d.o_tok_stride = 8          # rows that overlap: a view of less memory
    assert lib.animaxs_kv8_attn_validate(None, ctypes.byref(c), ctypes.byref(d), 0x5000, 0x6000) == code


@pytest.mark.parametrize("capacity,code", [((1 << 31) - 65, 0), ((1 << 31) - 64, -8), ((1 << 31) - 1, -8)])
def test_positions(lib, capacity, code):
    """Positions are numbered in 32 bits up to the end of the last block."""
    assert _write(lib, 1, capacity, 1, 16) == code
    a, b = ctypes.c_int64(), ctypes.c_int64()
    assert lib.animaxs_kv8_cache_bytes(1, capacity, 1, 64, ctypes.byref(a), ctypes.byref(b)) == code


@pytest.mark.parametrize("offset,code", [(0, 0), (4, 0), (1, -1), (2, -1)])
def test_device_integers_are_aligned(lib, offset, code):
    """starts, counts and lengths are read as int32: an address between two of them is refused, not read."""
    from animaxs_b200._lib import AttnDesc, Kv8Cache, Kv8WriteDesc
    c = Kv8Cache(1, 512, 1, 64, 0, 0x1000, 0x2000, 0x3000, 0x4000)
    for name in ("starts", "counts"):
        w = Kv8WriteDesc(16, 0, None, None, 64, 64, 1024, 64, 64, 1024)
        setattr(w, name, 0x7000 + offset)
        assert lib.animaxs_kv8_write_validate(None, ctypes.byref(c), ctypes.byref(w), 0x5000, 0x6000) == code
    d = AttnDesc()
    lib.animaxs_attn_desc_init(ctypes.byref(d), 1, 1, 1, 3, 512, 64)
    d.kv_valid_lens = 0x7000 + offset
    assert lib.animaxs_kv8_attn_validate(None, ctypes.byref(c), ctypes.byref(d), 0x5000, 0x6000) == code
