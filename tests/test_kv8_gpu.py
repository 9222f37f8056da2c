"""GPU: the 8-bit K/V cache -- written codes and scales against the definition's arithmetic, bit for bit, read-back
and attention against float64.

Attention's tolerance: the output is rounded to fp16 (2^-11 of itself); each probability is rounded to fp16 relative
to a maximum that may lag by 2^8 (2^-11 of itself, or 2^-25 absolutely where it is subnormal, for each of the N
keys), and exp2 and the fp32 scores add less than 2^-12.  So |out - ref| <= 2^-10 |ref| + (2^-10 + N 2^-25) max|v|."""
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


def _cache(ex, fmt, batch, capacity, heads, dim, seed=0, garbage=True):
    """A cache whose buffers hold arbitrary bytes (NaN codes and scales among them)."""
    import torch

    from animaxs_b200 import QuantizedKVCache
    c = QuantizedKVCache(ex, batch=batch, capacity=capacity, kv_heads=heads, head_dim=dim, format=fmt)
    if garbage:
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (c.k_codes, c.v_codes):
            t.view(torch.uint8).random_(0, 256, generator=g)
        for t in (c.k_scale, c.v_scale):
            t.fill_(float("nan"))
    return c


def _values(codes):
    return codes.double().cpu().numpy()


def _rand(g, shape, outliers=False):
    x = g.standard_normal(shape)
    if outliers:
        x[..., ::17] *= 6
    return x.astype(np.float16)


def _dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _ints(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _check_write(cache, state, k, v, starts, counts, fmt):
    """Apply the oracle to ``state`` (values and scales per tensor) and compare what lies before each sequence's end."""
    for name, x in (("k", k), ("v", v)):
        values, scale = state[name]
        got_v, got_s = _values(getattr(cache, name + "_codes")), getattr(cache, name + "_scale").cpu().numpy()
        for b in range(cache.batch):
            for h in range(cache.kv_heads):
                values[b, h], scale[b, h] = ora.write(values[b, h], scale[b, h], x[b, :, h], fmt, starts[b], counts[b])
                end = min(cache.capacity, max(starts[b], 0) if counts[b] <= 0 else starts[b] + min(counts[b], x.shape[1]))
                n = max(end, 0)
                assert np.array_equal(got_v[b, h, :n], values[b, h, :n], equal_nan=True), (name, b, h)
                blocks = -(-n // 64)
                assert np.array_equal(got_s[b, h, :blocks], scale[b, h, :blocks], equal_nan=True), (name, b, h)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("batch,tokens,heads,dim,capacity,starts", [
    (1, 1, 1, 64, 1, [0]), (2, 1, 8, 128, 130, [0, 63]), (3, 64, 2, 128, 200, [0, 64, 1]),
    (2, 65, 3, 64, 129, [0, 64]), (2, 200, 2, 128, 333, [0, 127]), (1, 129, 16, 128, 512, [300])])
def test_write_is_the_definition(ex, fmt, batch, tokens, heads, dim, capacity, starts):
    """A first write at 0 up to each start, then the write under test behind it."""
    import torch
    g = np.random.default_rng(tokens + dim)
    cache = _cache(ex, fmt, batch, capacity, heads, dim)
    state = {n: (_values(getattr(cache, n + "_codes")), getattr(cache, n + "_scale").cpu().numpy()) for n in "kv"}
    if max(starts) > 0:
        k, v = (_rand(g, (batch, max(starts), heads, dim)) * np.float16(0.25) for _ in range(2))
        cache.write(_dev(k), _dev(v), counts=_ints(starts))
        _check_write(cache, state, k, v, [0] * batch, starts, fmt)
    # K and V as the column halves of one projection's rows.
    rows = _rand(g, (batch, tokens, 2, heads, dim), outliers=True)
    dev = _dev(rows)
    cache.write(dev[:, :, 0], dev[:, :, 1], starts=_ints(starts))
    _check_write(cache, state, rows[:, :, 0], rows[:, :, 1], starts, [tokens] * batch, fmt)
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    cache.write(dev[:, :, 0], dev[:, :, 1], starts=_ints(starts))   # repeating it changes nothing
    for a, t in zip(before, (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)):
        assert torch.equal(a.view(torch.uint8), t.view(torch.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
def test_appending_token_by_token(ex, fmt):
    """150 appends with growing values: the block's scale grows and older codes are re-rounded each time."""
    g = np.random.default_rng(5)
    cache = _cache(ex, fmt, 2, 160, 2, 128)
    state = {n: (_values(getattr(cache, n + "_codes")), getattr(cache, n + "_scale").cpu().numpy()) for n in "kv"}
    for t in range(150):
        k, v = (_rand(g, (2, 1, 2, 128)) * np.float16(0.1 + 0.01 * t) for _ in range(2))
        cache.write(_dev(k), _dev(v), t)
        if t in (0, 1, 62, 63, 64, 127, 128, 149):
            _check_write(cache, state, k, v, [t, t], [1, 1], fmt)
        else:
            for n, x in (("k", k), ("v", v)):
                for b in range(2):
                    for h in range(2):
                        state[n][0][b, h], state[n][1][b, h] = ora.write(state[n][0][b, h], state[n][1][b, h],
                                                                         x[b, :, h], fmt, t, 1)


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_edges(ex, fmt):
    """Counts of zero, past the rows and negative; positions before 0 and past the capacity; zeros, infinities, NaN,
    the largest and the smallest fp16."""
    g = np.random.default_rng(9)
    cache = _cache(ex, fmt, 5, 100, 1, 64)
    state = {n: (_values(getattr(cache, n + "_codes")), getattr(cache, n + "_scale").cpu().numpy()) for n in "kv"}
    untouched = cache.k_codes[0].clone()
    k, v = _rand(g, (5, 40, 1, 64)), np.zeros((5, 40, 1, 64), np.float16)
    k[2, 3, 0, 5], k[2, 4, 0, 6], k[2, 5, 0, 7] = np.inf, -np.inf, np.nan
    k[3, :, 0, :] = np.float16(6e-8)
    k[4, 7, 0, 1] = 65504
    v[2, 9, 0, 3] = np.inf                                   # among zeros: the scale stays 0
    starts, counts = [0, 80, -3, 0, 0], [-2, 40, 39, 99, 40]
    cache.write(_dev(k), _dev(v), starts=_ints(starts), counts=_ints(counts))
    _check_write(cache, state, k, v, starts, [min(c, 40) for c in counts], fmt)
    import torch
    assert torch.equal(cache.k_codes[0].view(torch.uint8), untouched.view(torch.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,start,tokens,lens", [(128, 0, 200, None), (64, 37, 101, [90, 138]), (128, 199, 1, [0, 200])])
def test_read(ex, fmt, dim, start, tokens, lens):
    """fp16(code * scale), one rounding: half a unit in the last place of the float64 product (and fp32's 2^-24)."""
    import torch
    g = np.random.default_rng(2)
    cache = _cache(ex, fmt, 2, 200, 3, dim)
    k, v = (_rand(g, (2, 200, 3, dim), outliers=True) for _ in range(2))
    cache.write(_dev(k), _dev(v))
    wide = torch.full((2, tokens, 8, dim), 7.0, dtype=torch.float16, device="cuda")
    vw = wide.clone()
    got = cache.read(start, tokens, lens=None if lens is None else _ints(lens), k_out=wide[:, :, 2:5], v_out=vw[:, :, 2:5])
    for name, out in zip("kv", got):
        want = ora.decode(_values(getattr(cache, name + "_codes")), getattr(cache, name + "_scale").cpu().numpy())
        want = want.transpose(0, 2, 1, 3)[:, start:start + tokens].copy()
        for b in range(2):
            if lens is not None:
                want[b, max(0, lens[b] - start):] = 0
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all()
    assert (wide[:, :, :2] == 7).all() and (wide[:, :, 5:] == 7).all()
    # An int8 round trip is off by at most half a step (and the read's own rounding).
    if fmt == "int8" and lens is None:
        step = np.repeat(cache.k_scale.cpu().numpy(), 64, axis=-1)[:, :, :200].transpose(0, 2, 1)[..., None]
        full = k.astype(np.float64)[:, start:start + tokens]
        assert (np.abs(got[0].double().cpu().numpy() - full) <= 0.5001 * step + np.abs(full) * 2.0 ** -10).all()


def _attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal=False, kv_len=None, seed=0, scale=None,
            q=None, mutate=None):
    """(out, reference, bound) of one attention call over a freshly written cache."""
    import torch
    g = np.random.default_rng(seed + 13)
    cache = _cache(ex, fmt, batch, capacity, kv_heads, dim)
    most = max(max(lens), 1)
    k, v = _rand(g, (batch, most, kv_heads, dim), outliers=True), _rand(g, (batch, most, kv_heads, dim))
    if mutate is not None:
        mutate(k, v)
    cache.write(_dev(k), _dev(v), counts=_ints(lens))
    if q is None:
        q = _rand(g, (batch, q_len, heads, dim))
    out = cache.attention(_dev(q), lens=_ints(lens), causal=causal, kv_len=kv_len, scale=scale)
    ex.synchronize(torch.cuda.current_stream())
    kd = ora.decode(np.nan_to_num(_values(cache.k_codes)), np.nan_to_num(cache.k_scale.cpu().numpy()))
    vd = ora.decode(np.nan_to_num(_values(cache.v_codes)), np.nan_to_num(cache.v_scale.cpu().numpy()))
    ref = ora.attention(q, kd, vd, lens, causal, scale)
    vmax = np.array([np.abs(vd[b, :, :max(n, 1)]).max() for b, n in enumerate(lens)])[:, None, None, None]
    bound = 2.0 ** -10 * np.abs(ref) + (2.0 ** -10 + max(lens) * 2.0 ** -25) * vmax
    return out.double().cpu().numpy(), ref, bound


def _assert_close(got, ref, bound):
    assert np.isfinite(got).all()
    err = np.abs(got - ref)
    assert (err <= bound).all(), f"worst {np.max(err / bound):.2f} of the bound"


FEW = [  # batch, q_len, heads, kv_heads, dim, capacity, lens, causal
    (1, 1, 1, 1, 128, 1, [1], False),
    (1, 1, 16, 8, 128, 512, [300], False),
    (3, 1, 16, 8, 128, 700, [1, 64, 65], True),
    (4, 1, 8, 8, 64, 500, [63, 0, 500, 129], False),
    (2, 5, 16, 16, 64, 300, [3, 257], True),          # more queries than tokens: the first see nothing
    (2, 16, 2, 2, 128, 200, [200, 100], True),
    (1, 1, 16, 1, 128, 5000, [4999], False),          # 16 rows, one line over all CTAs
    (2, 2, 14, 2, 128, 1000, [999, 130], True),       # a group of 7
    (40, 1, 4, 2, 128, 300, [(37 * i) % 301 for i in range(40)], False),
    (150, 1, 2, 1, 64, 130, [(i * 7) % 131 for i in range(150)], False),   # more sequences than the scan's shares
    (5, 1, 2, 2, 128, 64, [0, 0, 0, 0, 0], False),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", FEW, ids=[str(i) for i in range(len(FEW))])
def test_attention_few_rows(ex, fmt, case):
    batch, q_len, heads, kv_heads, dim, capacity, lens, causal = case
    got, ref, bound = _attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal)
    _assert_close(got, ref, bound)


# How a line's keys are shared out follows from the number of lines and the longest one they may have.
SHARES = [  # batch, q_len, heads, kv_heads, dim, capacity, lens, causal
    (1, 1, 2, 1, 128, 1600, [1600], False),           # a cluster of CTAs to a line
    (2, 3, 8, 4, 128, 1100, [1100, 37], True),
    (4, 1, 8, 4, 64, 1000, [1000, 0, 33, 512], False),
    (3, 2, 24, 8, 128, 700, [700, 31, 65], True),
    (9, 1, 16, 8, 64, 500, [(61 * i) % 501 for i in range(9)], False),
    (1, 1, 16, 1, 128, 12000, [11999], False),        # equal shares: one line over all CTAs
    (2, 4, 8, 4, 64, 9000, [9000, 70], True),
    (3, 1, 16, 8, 128, 8000, [8000, 1, 4001], False),
    (2, 1, 16, 8, 128, 7000, [300, 0], False),        # lines that turn out short: a CTA to each
    (3, 2, 12, 6, 128, 9000, [96, 700, 1], True),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", SHARES, ids=[str(i) for i in range(len(SHARES))])
def test_attention_few_rows_shares(ex, fmt, case):
    batch, q_len, heads, kv_heads, dim, capacity, lens, causal = case
    got, ref, bound = _attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal)
    _assert_close(got, ref, bound)


MANY = [
    (1, 17, 1, 1, 128, 64, [40], False),
    (1, 128, 2, 1, 128, 128, [128], False),
    (2, 129, 4, 2, 128, 300, [300, 1], True),
    (2, 300, 2, 2, 64, 515, [513, 47], False),
    (3, 257, 6, 2, 128, 400, [400, 0, 129], True),    # a group of 3; a sequence without tokens
    (1, 200, 14, 2, 64, 300, [100], True),            # a group of 7, more queries than tokens
    (1, 1024, 16, 16, 128, 512, [128], False),        # an image's queries on a padded context
    (1, 64, 16, 8, 128, 3000, [2999], True),          # a prompt chunk on a long cache
    (2, 40, 32, 2, 128, 1000, [1000, 321], True),     # a group of 16
    (5, 300, 10, 10, 64, 2000, [2000, 0, 1999, 65, 700], True),   # equal shares of the keys over all SMs
    (3, 290, 40, 20, 128, 1500, [1500, 1, 833], False),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", MANY, ids=[str(i) for i in range(len(MANY))])
def test_attention_many_rows(ex, fmt, case):
    batch, q_len, heads, kv_heads, dim, capacity, lens, causal = case
    got, ref, bound = _attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity, lens, causal)
    _assert_close(got, ref, bound)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("q_len", [1, 140])
def test_attention_scales_of_every_size(ex, fmt, q_len):
    """Blocks of values a million times smaller or larger than their neighbours, and blocks of zeros."""
    def mutate(k, v):
        v[:, 0:64] *= np.float16(1e-4)
        v[:, 64:128] = 0
        v[:, 128:192] *= np.float16(100)
        k[:, 192:256] = 0
        k[:, 0:64] *= np.float16(4)
    got, ref, bound = _attend(ex, fmt, 2, q_len, 4, 2, 128, 400, [400, 256], mutate=mutate)
    _assert_close(got, ref, bound)


@pytest.mark.parametrize("q_len", [1, 140])
def test_attention_all_values_zero_or_tiny(ex, q_len):
    def zero(k, v):
        v[:] = 0
    got, _, _ = _attend(ex, "int8", 1, q_len, 4, 2, 64, 200, [200], mutate=zero)
    assert (got == 0).all()

    def tiny(k, v):
        v[:] = np.float16(6e-8)                               # fp16's smallest: the output is that value
    got, ref, _ = _attend(ex, "int8", 1, q_len, 4, 2, 64, 200, [200], mutate=tiny)
    assert np.array_equal(got, np.full_like(got, np.float64(np.float16(6e-8))))


@pytest.mark.parametrize("q_len", [1, 150])
def test_attention_large_scores(ex, q_len):
    """Scores of hundreds: one key takes everything, and the running maximum has to follow through all tiles."""
    def rising(k, v):
        k[:] = (np.linspace(0.1, 8, k.shape[1])[None, :, None, None] * np.sign(k)).astype(np.float16)
    got, ref, bound = _attend(ex, "int8", 1, q_len, 2, 2, 128, 700, [700], mutate=rising, scale=1.5)
    # The scores' own fp32 rounding counts here: |s| <= 1.5 * 128 * 8 * 4 = 6144, off by up to 6144 * 2^-22.
    _assert_close(got, ref, bound + 6144 * 2.0 ** -21 * np.abs(ref).max())


@pytest.mark.parametrize("q_len", [1, 150])
def test_attention_nan_queries_stay_in_their_rows(ex, q_len):
    g = np.random.default_rng(3)
    q = _rand(g, (2, q_len, 4, 128))
    q[1, 0, 2, 5] = np.nan
    got, ref, bound = _attend(ex, "int8", 2, q_len, 4, 2, 128, 200, [200, 77], q=q)
    assert np.isnan(got[1, 0, 2]).all()
    ref[1, 0, 2], got[1, 0, 2], bound[1, 0, 2] = 0, 0, 1
    _assert_close(got, ref, bound)


@pytest.mark.parametrize("q_len,kv_len", [(1, 700), (1, 4000), (6, 4000), (1, 15000), (200, 1500)])
def test_attention_is_repeatable_and_uses_its_stream(ex, q_len, kv_len):
    """The same bits on every call (split keys are joined in a fixed order), on another stream, into a strided output."""
    import torch
    g = np.random.default_rng(1)
    cache = _cache(ex, "int8", 2, kv_len, 2, 128)
    k, v = (_dev(_rand(g, (2, kv_len, 2, 128))) for _ in range(2))
    lens = _ints([kv_len, kv_len // 3])
    q = _dev(_rand(g, (2, q_len, 4, 128)))
    cache.write(k, v)
    first = cache.attention(q, lens=lens)
    for _ in range(5):
        assert torch.equal(cache.attention(q, lens=lens), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    wide = torch.full((2, q_len, 4, 256), 3.0, dtype=torch.float16, device="cuda")
    heads = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)     # head-major
    side.wait_stream(torch.cuda.current_stream())
    cache.attention(heads, wide[..., 128:], lens=lens, stream=side)
    side.synchronize()
    assert torch.equal(wide[..., 128:], first) and (wide[..., :128] == 3).all()


@pytest.mark.parametrize("batch,q_len,heads,kv_heads,dim,kv_len,causal", [
    (2, 1700, 16, 8, 64, 378, False), (1, 600, 16, 16, 128, 2000, False), (3, 294, 16, 8, 64, 648, True),
    (20, 1, 16, 8, 128, 1500, True), (4, 8, 4, 2, 64, 2000, False)])
def test_attention_many_calls_agree(ex, batch, q_len, heads, kv_heads, dim, kv_len, causal):
    """Bit for bit over 400 calls: a copy that overtook the readers of its shared-memory slot would show here."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = _cache(ex, "e4m3", batch, kv_len, kv_heads, dim)
    k, v = (torch.randn((batch, kv_len, kv_heads, dim), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((batch, q_len, heads, dim), generator=g, device="cuda").half()
    cache.write(k, v)
    outs = [cache.attention(q, causal=causal) for _ in range(2)]
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(400):
        cache.attention(q, outs[1], causal=causal)
        differ += (outs[1].view(torch.int16) != outs[0].view(torch.int16)).any()
    assert int(differ) == 0


def test_positions_past_32_bits(ex):
    """Codes beyond 4 GiB of a buffer: the third sequence of three of 18 million tokens, and its last block."""
    import torch
    g = np.random.default_rng(6)
    cap = 18_000_000
    cache = _cache(ex, "int8", 3, cap, 1, 128, garbage=False)
    k, v = (_rand(g, (3, 300, 1, 128)) for _ in range(2))
    cache.write(_dev(k), _dev(v))
    q = _rand(g, (3, 4, 2, 128))
    lens = [0, 17, 300]
    many = _rand(g, (3, 70, 2, 128))
    for queries in (q, many):
        out = cache.attention(_dev(queries), lens=_ints(lens), causal=True)
        kd = ora.decode(_values(cache.k_codes[:, :, :300]), cache.k_scale[:, :, :5].cpu().numpy())
        vd = ora.decode(_values(cache.v_codes[:, :, :300]), cache.v_scale[:, :, :5].cpu().numpy())
        ref = ora.attention(queries, kd, vd, lens, True)
        bound = 2.0 ** -10 * np.abs(ref) + (2.0 ** -10 + 300 * 2.0 ** -25) * np.abs(vd).max()
        _assert_close(out.double().cpu().numpy(), ref, bound)
    cache.write(_dev(k), _dev(v), cap - 300)
    rk, rv = cache.read(cap - 300, 300)
    for got, x in ((rk, k), (rv, v)):
        err = np.abs(got.double().cpu().numpy() - x.astype(np.float64))
        assert (err <= np.abs(x).max() / 127 * 0.51 + np.abs(x) * 2.0 ** -10).all()
    assert torch.equal(cache.read(cap - 1, 1)[0], rk[:, -1:])


def test_attention_normalises_q(ex):
    """qk_norm="rms" is the attention prologue's normalisation followed by the plain call."""
    import torch
    g = np.random.default_rng(8)
    cache = _cache(ex, "int8", 2, 300, 16, 128)
    cache.write(_dev(_rand(g, (2, 300, 16, 128))), _dev(_rand(g, (2, 300, 16, 128))))
    q = _dev(_rand(g, (2, 50, 16, 128)) * np.float16(3))
    w = _dev((1 + 0.2 * g.standard_normal(128)).astype(np.float16))
    normed = torch.empty_like(q)
    ex.rmsnorm_heads_half(torch.cuda.current_stream(), q, normed, w, tokens=100, heads=16)
    assert torch.equal(cache.attention(q, qk_norm="rms", q_norm_weight=w), cache.attention(normed))


def test_python_refusals(ex):
    import torch

    from animaxs_b200 import AttentionValidationError, QuantizedKVCache
    cache = _cache(ex, "int8", 2, 100, 4, 64)
    h = torch.zeros((2, 10, 4, 64), dtype=torch.float16, device="cuda")
    bad = [
        lambda: QuantizedKVCache(ex, head_dim=96),
        lambda: QuantizedKVCache(ex, format="int4"),
        lambda: QuantizedKVCache.wrap(ex, cache.k_codes.float(), cache.v_codes, cache.k_scale, cache.v_scale),
        lambda: QuantizedKVCache.wrap(ex, cache.k_codes, cache.v_codes, cache.k_scale[..., :1], cache.v_scale),
        lambda: QuantizedKVCache.wrap(ex, cache.k_codes.transpose(0, 1), cache.v_codes.transpose(0, 1), cache.k_scale,
                                      cache.v_scale),
        lambda: cache.write(h.float(), h.float()),
        lambda: cache.write(h, h[:, :9]),
        lambda: cache.write(h[:, :, :3], h[:, :, :3]),
        lambda: cache.write(h, h, 95),
        lambda: cache.write(h, h, starts=torch.zeros(2, dtype=torch.int64, device="cuda")),
        lambda: cache.write(h, h, counts=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: cache.read(95, 10),
        lambda: cache.attention(h[:, :, :3]),
        lambda: cache.attention(h, kv_len=101),
        lambda: cache.attention(h.bfloat16()),
        lambda: cache.attention(h, qk_norm="rms_rope"),
        lambda: cache.attention(h, h[:, :5]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AttentionValidationError):
            call()
            pytest.fail(f"call {i} was accepted")
