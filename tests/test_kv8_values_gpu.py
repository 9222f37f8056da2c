"""GPU: attention over 8-bit caches of arbitrary content, as a caller's own buffers may hold it, against float64.

Bounds per element as for written caches: |out - ref| <= 2^-10 |ref| + (2^-10 + N 2^-25) max|v|: fp16 output, fp16
probabilities relative to a maximum that may lag by 2^8, fp32 scores."""
import numpy as np
import pytest

from oracle import kv8_oracle as ora

pytestmark = pytest.mark.gpu
FORMATS = ["int8", "e4m3"]


@pytest.fixture(scope="module")
def ex():
    from animaxs_b200 import AttentionExecutor
    e = AttentionExecutor(0)
    yield e
    e.close()


def _wrapped(ex, fmt, batch, kv_heads, tokens, dim, seed):
    """Random codes under random scales, made on the host; (cache, K, V as float64)."""
    import torch

    from animaxs_b200 import QuantizedKVCache
    g = np.random.default_rng(seed)
    tensors, decoded = [], []
    for top in (0.02, 0.01):
        codes = g.integers(-127, 128, (batch, kv_heads, tokens, dim)).astype(np.float32)
        codes = torch.from_numpy(codes).to(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
        scale = (top * g.uniform(0.2, 1, (batch, kv_heads, -(-tokens // 64)))).astype(np.float32)
        scale[:, :, 1::3] = 0
        tensors.append((codes.cuda(), torch.from_numpy(scale).cuda()))
        decoded.append(ora.decode(codes.double().numpy(), scale))
    (kc, ks), (vc, vs) = tensors
    return QuantizedKVCache.wrap(ex, kc, vc, ks, vs), *decoded


def _check(got, ref, v, keys):
    bound = 2.0 ** -10 * np.abs(ref) + (2.0 ** -10 + keys * 2.0 ** -25) * np.abs(v).max()
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= bound).all(), f"worst {np.max(err / bound):.2f} of the bound"


SHAPES = [(1, 1, 4, 2, 128, 300), (2, 3, 6, 2, 64, 200), (1, 1, 2, 1, 128, 12000),   # few rows: alone, shared, split
          (2, 40, 4, 2, 128, 400), (1, 300, 3, 1, 64, 700), (2, 150, 8, 8, 128, 130)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_a_scale_of_zero_makes_values_of_zero(ex, fmt, shape):
    """Every third block's scale is 0 under codes that are not: its keys score 0 and its values are 0."""
    import torch
    batch, q_len, heads, kv_heads, dim, keys = shape
    cache, k, v = _wrapped(ex, fmt, batch, kv_heads, keys, dim, keys)
    q = np.random.default_rng(keys + 1).standard_normal((batch, q_len, heads, dim)).astype(np.float16)
    lens = [keys - 45 * i for i in range(batch)]
    out = cache.attention(torch.from_numpy(q).cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          causal=True)
    _check(out, ora.attention(q, k, v, lens, True), v, keys)
    rk, rv = cache.read()
    for got, x in ((rk, k), (rv, v)):
        assert (got.cpu().numpy()[:, 64:128][np.abs(x.transpose(0, 2, 1, 3)[:, 64:128]) == 0] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("scale", [1e-38, 1e-44])
def test_a_softmax_scale_that_underflows(ex, fmt, shape, scale):
    """A scale so small that its product with a block's vanishes: every visible key weighs the same, masked ones
    nothing."""
    import torch
    batch, q_len, heads, kv_heads, dim, keys = shape
    cache, k, v = _wrapped(ex, fmt, batch, kv_heads, keys, dim, keys)
    q = np.random.default_rng(keys + 1).standard_normal((batch, q_len, heads, dim)).astype(np.float16)
    lens = [keys - 45 * i for i in range(batch)]
    out = cache.attention(torch.from_numpy(q).cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          causal=True, scale=scale)
    _check(out, ora.attention(q, k, v, lens, True, scale), v, keys)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_write_of_more_tokens_than_the_capacity(ex, fmt):
    """5000 tokens of which the last 50 and 120 fall inside a cache of 100: codes and scales are the definition's."""
    import torch

    from animaxs_b200 import QuantizedKVCache
    x = np.random.default_rng(3).standard_normal((2, 5000, 2, 64)).astype(np.float16)
    cache = QuantizedKVCache(ex, batch=2, capacity=100, kv_heads=2, head_dim=64, format=fmt)
    starts = [-4950, -4880]
    dev = torch.from_numpy(x).cuda()
    cache.write(dev, dev, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    for b in range(2):
        for h in range(2):
            values, scale = ora.write(np.zeros((100, 64)), np.zeros(2, np.float32), x[b, :, h], fmt, starts[b], 5000)
            for codes, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
                assert np.array_equal(codes[b, h].double().cpu().numpy(), values)
                assert np.array_equal(s[b, h].cpu().numpy(), scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("tiny", [1e-20, 1e-30, 2e-38, 1e-38, 1e-40, 1e-45])
def test_a_v_scale_that_makes_values_vanish(ex, fmt, shape, tiny):
    """Blocks of zeros often come with the least scale that a quantiser divides by (fp32's least normal / 127, say):
    their values add nothing that fp16 holds, but their keys keep their weights."""
    import torch
    batch, q_len, heads, kv_heads, dim, keys = shape
    cache, k, v = _wrapped(ex, fmt, batch, kv_heads, keys, dim, keys)
    blocks = cache.v_scale.shape[2]
    cache.v_scale[:, :, 0::2] = tiny
    if blocks > 1:
        cache.v_scale[:, :, 1::2] = 0.01
    v = ora.decode(cache.v_codes.double().cpu().numpy(), cache.v_scale.cpu().numpy())
    q = np.random.default_rng(keys + 1).standard_normal((batch, q_len, heads, dim)).astype(np.float16)
    lens = [keys - 45 * i for i in range(batch)]
    out = cache.attention(torch.from_numpy(q).cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          causal=True)
    _check(out, ora.attention(q, k, v, lens, True), v, keys)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [1e-38, 1e-39, 1e-45])
def test_zeros_behind_a_vanishing_scale(ex, fmt, scale):
    """Tokens of zeros appended to a block whose scale is so small that its inverse overflows: codes of 0, the older
    ones and the scale as they were; values that are not zero take the scale over."""
    import torch

    from animaxs_b200 import QuantizedKVCache
    cache = QuantizedKVCache(ex, batch=1, capacity=128, kv_heads=2, head_dim=64, format=fmt)
    for codes, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        codes[:, :, :10].copy_(torch.full((1, 2, 10, 64), 3.0, device="cuda").to(codes.dtype))
        codes[:, :, 10:].view(torch.uint8).fill_(0x55)
        s.fill_(scale)
    held = cache.k_scale.clone()
    zeros = torch.zeros((1, 20, 2, 64), dtype=torch.float16, device="cuda")
    cache.write(zeros, zeros, 10)
    for codes, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        assert (codes[:, :, 10:30].float() == 0).all() and (codes[:, :, :10].float() == 3).all()
        assert torch.equal(s, held)
    ones = torch.ones((1, 1, 2, 64), dtype=torch.float16, device="cuda")
    cache.write(ones, ones, 30)
    top = 127 if fmt == "int8" else 448
    assert (cache.k_codes[:, :, 30].float() == top).all() and (cache.k_codes[:, :, :30].float() == 0).all()
