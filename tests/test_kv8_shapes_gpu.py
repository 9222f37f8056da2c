"""GPU: attention over the 8-bit cache, whole outputs against float64, at the shapes where rows and lines are laid out
differently.

Besides the element bound, whose N 2^-25 max|v| hides a lost tile of a long line, each (sequence, head)'s output is
held to 1e-3 of its norm.  Rounding to fp16 once at the end and once in the probabilities are errors of up to 2^-11 of
each value, uniform in it: 2^-11 / sqrt(3) = 2.8e-4 each in the norm, 4.0e-4 together, and up to 2^-12 more from exp2
and the fp32 scores.  One 32-key tile left out of 12000 keys moves it by 4e-2."""
import numpy as np
import pytest

from test_kv8_gpu import FEW, FORMATS, MANY, SHARES, _assert_close, _attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    from animaxs_b200 import AttentionExecutor
    e = AttentionExecutor(0)
    yield e
    e.close()


def _check(got, ref, bound):
    _assert_close(got, ref, bound)
    err, norm = (np.sqrt((x ** 2).sum(axis=(1, 3))) for x in (got - ref, ref))   # [batch, heads]
    assert (err[norm == 0] == 0).all()
    assert (err <= 1e-3 * norm).all(), f"worst {np.max(err[norm > 0] / norm[norm > 0]):.2e} of the norm"


CASES = [(n, i, c) for n, cases in (("few", FEW), ("shares", SHARES), ("many", MANY)) for i, c in enumerate(cases)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", [c for _, _, c in CASES], ids=[f"{n}{i}" for n, i, _ in CASES])
def test_norm(ex, fmt, case):
    batch, q_len, heads, kv_heads, dim, capacity, lens, causal = case
    _check(*_attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal))


BATCHES = [  # batch, q_len, heads, kv_heads, dim, capacity, lens, causal: more than 256 sequences
    (257, 1, 2, 1, 64, 130, [(i * 7) % 131 for i in range(257)], False),
    (600, 1, 4, 2, 128, 200, [(i * 61) % 201 if i % 5 else 0 for i in range(600)], False),
    (600, 3, 2, 2, 64, 100, [(i * 13) % 101 for i in range(600)], True),
    (513, 1, 1, 1, 128, 900, [900 if i in (0, 200, 512) else i % 3 for i in range(513)], False),
    (300, 2, 6, 3, 64, 90, [0] * 299 + [90], True),
    (1030, 1, 2, 2, 64, 64, [0 if i < 700 else 64 for i in range(1030)], False),
    (260, 20, 2, 1, 64, 130, [(i * 7) % 131 for i in range(260)], True),      # many rows
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", BATCHES, ids=[str(i) for i in range(len(BATCHES))])
def test_large_batches(ex, fmt, case):
    """Sequences in groups of two and more in the search for a tile's place, empty ones among them."""
    batch, q_len, heads, kv_heads, dim, capacity, lens, causal = case
    _check(*_attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal))


GROUPS = [  # heads / kv_heads of 16 rows and more: 32-row boxes hold some of a token's heads
    (2, 1, 32, 2, 128, 16, 300, [300, 77], False),
    (1, 1, 32, 1, 128, 32, 200, [199], False), (2, 5, 64, 2, 64, 32, 300, [300, 2], True),
    (1, 1, 64, 1, 64, 64, 130, [130], False), (1, 9, 128, 2, 128, 64, 500, [500], True),
    (2, 1, 128, 1, 128, 128, 100, [100, 0], False), (1, 3, 128, 1, 64, 128, 2000, [1999], True),
    (1, 1, 256, 1, 64, 256, 90, [90], False), (1, 3, 256, 1, 128, 256, 130, [130], True),
    (1, 7, 48, 1, 64, 48, 300, [300], True),                                    # does not divide 128
    (3, 40, 192, 3, 64, 64, 200, [200, 31, 7], True), (2, 300, 64, 2, 128, 32, 100, [100, 64], False),
    (1, 2, 128, 1, 128, 128, 5000, [5000], False),                              # one line over all CTAs
    (20, 8, 32, 1, 64, 32, 400, [(i * 37) % 401 for i in range(20)], True),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", GROUPS, ids=[f"{c[5]}-{c[1]}" for c in GROUPS])
def test_large_groups(ex, fmt, case):
    batch, q_len, heads, kv_heads, dim, group, capacity, lens, causal = case
    assert heads == kv_heads * group
    _check(*_attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal))
