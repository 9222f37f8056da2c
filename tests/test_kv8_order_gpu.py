"""GPU: calls of the 8-bit K/V cache that follow one another on a stream see each other's results.

The kernels start while their predecessors end (programmatic dependent launch), so each pair here runs many times
without a synchronisation and is compared bit for bit with calls that the host waited for."""
import pytest

pytestmark = pytest.mark.gpu
FORMATS = ["int8", "e4m3"]


@pytest.fixture(scope="module")
def ex():
    from animaxs_b200 import AttentionExecutor
    e = AttentionExecutor(0)
    yield e
    e.close()


def _draw(seed, *shape):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").half()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("batch,q_len,heads,kv_heads,dim,capacity", [
    (1, 1, 8, 8, 128, 64), (4, 1, 16, 8, 64, 128), (3, 2, 4, 2, 128, 256), (2, 20, 8, 4, 64, 256),
    (1, 1, 6, 6, 128, 192)])
def test_append_then_attend(ex, fmt, batch, q_len, heads, kv_heads, dim, capacity):
    """400 steps of append, attention and read-back.  Capacities of a few blocks put the scales of several heads into
    one 32-byte sector, which other CTAs of the append write while one of them reads its own; values that grow
    from step to step make every append re-round its block and change its scale."""
    import torch

    from animaxs_b200 import QuantizedKVCache

    def run(wait):
        cache = QuantizedKVCache(ex, batch=batch, capacity=capacity, kv_heads=kv_heads, head_dim=dim, format=fmt)
        stream = torch.cuda.current_stream()
        outs, reads = [], []
        lens = torch.empty(batch, dtype=torch.int32, device="cuda")
        for i in range(400):
            at = i * q_len % (capacity - q_len + 1)
            x = i % steps
            lens.fill_(at + q_len)
            cache.write(k[x], v[x], at)
            if wait:
                ex.synchronize(stream)
            outs.append(cache.attention(q[x], lens=lens, causal=True))
            if wait:
                ex.synchronize(stream)
            if i % 40 == 39:
                reads.append(torch.stack(cache.read(tokens=at + q_len)))
        ex.synchronize(stream)
        return outs, reads

    steps = 40
    grow = torch.linspace(0.1, 3, steps, device="cuda").half()[:, None, None, None, None]
    k, v = (_draw(s, steps, batch, q_len, kv_heads, dim) * grow for s in (1, 2))
    q = _draw(3, steps, batch, q_len, heads, dim)
    want, got = run(True), run(False)
    for part in range(2):
        for i, (a, b) in enumerate(zip(want[part], got[part])):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), (part, i)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_then_attend_alone(ex, fmt):
    """The same with nothing between the two calls: positions and lengths stand on the device before the loop."""
    import torch

    from animaxs_b200 import QuantizedKVCache
    batch, kv_heads, dim, capacity = 2, 8, 128, 200
    k, v, q = (_draw(s, capacity, batch, 1, kv_heads, dim) for s in (4, 5, 6))
    ends = torch.arange(1, capacity + 1, dtype=torch.int32, device="cuda")[:, None].repeat(1, batch).contiguous()
    starts = (ends - 1).contiguous()
    outs = torch.empty((2, 2, capacity, batch, 1, kv_heads, dim), dtype=torch.float16, device="cuda")
    stream = torch.cuda.current_stream()
    for wait in (1, 0):
        for again in range(2):
            cache = QuantizedKVCache(ex, batch=batch, capacity=capacity, kv_heads=kv_heads, head_dim=dim, format=fmt)
            for i in range(capacity):
                cache.write(k[i], v[i], starts=starts[i])
                if wait:
                    ex.synchronize(stream)
                cache.attention(q[i], outs[wait, again, i], lens=ends[i])
                if wait:
                    ex.synchronize(stream)
    ex.synchronize(stream)
    for again in range(2):
        assert torch.equal(outs[0, again].view(torch.int16), outs[1, 0].view(torch.int16))
