"""GPU: the 8-bit K/V cache's operators together, as ``examples/quantized_kv_cache.py`` runs them.

Bounds, with |k|, |v| < 6 (normalised or normal draws).  int8: a value written at once is off by half a step, 6 / 254
< 0.024; in a block that grew token by token each growth of the scale rounds again, by half a step of either sign,
taken as four steps (0.19) in all.  e4m3: half of a mantissa's 2^-3 at [4, 8), 0.25, and 0.375 with the scale's own
rounding; four times that for a grown block.  An output averages V under weights that the scores' error shifts; it is
held to 0.25 and 1.0: a wrong position, scale or mask moves outputs by several units at these lengths."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "quantized_kv_cache.py")
    spec = importlib.util.spec_from_file_location("example_quantized_kv_cache", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def ex():
    from animaxs_b200 import AttentionExecutor
    e = AttentionExecutor(0)
    yield e
    e.close()


@pytest.mark.parametrize("fmt,value,output", [("int8", 0.024, 0.25), ("e4m3", 0.375, 1.0)])
def test_cross_attention(example, ex, fmt, value, output):
    r = example.cross_attention(ex, blocks=2, steps=2, images=2, tokens=256, context=200, heads=4, format=fmt)
    assert r["value_difference"] <= value and r["output_difference"] <= output
    assert r["bytes"] < 0.51 * r["fp16_bytes"]


@pytest.mark.parametrize("fmt,value,output", [("int8", 0.19, 0.25), ("e4m3", 1.5, 1.0)])
def test_decode(example, ex, fmt, value, output):
    r = example.decode(ex, prompts=(150, 65, 1, 64), steps=20, chunk=64, heads=4, kv_heads=2, format=fmt)
    assert r["lengths"] == [170, 85, 21, 84]
    assert r["value_difference"] <= value and r["output_difference"] <= output
