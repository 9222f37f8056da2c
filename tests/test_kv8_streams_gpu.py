"""GPU: the 8-bit K/V cache's work on streams and in graphs -- what a captured step points at stays alive and is
put back, and steps that follow one another see each other's results.

Every comparison is bit for bit: equal calls give equal bits."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ex():
    """An executor of its own for each test: its workspaces are made by the test."""
    from animaxs_b200 import AttentionExecutor
    e = AttentionExecutor(0)
    yield e
    e.close()


def _draw(seed, *shape):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").half()


def _filled(ex, seed, batch, tokens, kv_heads, dim, fmt="int8", capacity=None):
    from animaxs_b200 import QuantizedKVCache
    c = QuantizedKVCache(ex, batch=batch, capacity=capacity or tokens, kv_heads=kv_heads, head_dim=dim, format=fmt)
    c.write(_draw(seed, batch, tokens, kv_heads, dim), _draw(seed + 1, batch, tokens, kv_heads, dim))
    return c


def _capture(call):
    """``call`` once on a side stream, then captured; returns the graph."""
    import torch
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


def _decoding_step(ex):
    """An append and an attention whose keys go to all SMs in equal shares; (call, output)."""
    import torch
    cache = _filled(ex, 1, 2, 4000, 4, 128, capacity=8000)
    k, v, q = _draw(3, 2, 1, 4, 128), _draw(4, 2, 1, 4, 128), _draw(5, 2, 1, 8, 128)
    at = torch.tensor([4000, 3333], dtype=torch.int32, device="cuda")
    lens, out = at + 1, torch.zeros_like(q)

    def step():
        cache.write(k, v, starts=at)
        cache.attention(q, out, lens=lens)
    return step, out


def test_a_graph_outlives_larger_calls(ex):
    """A decoding step captured first, replayed after calls that need the many-row workspace, more (sequence, head)
    lines than any call before, and one after the other of both: the same bits, and right ones for the others."""
    import torch
    step, out = _decoding_step(ex)
    graph = _capture(step)
    graph.replay()
    first = out.clone()
    chunk = _filled(ex, 7, 2, 3000, 4, 128)                    # 64 queries on 3000 keys: split over the CTAs
    queries = _draw(9, 2, 64, 8, 128)
    whole = chunk.attention(queries, causal=True)
    lines = _filled(ex, 11, 2100, 70, 8, 64)                   # 16800 lines
    token = _draw(13, 2100, 1, 8, 64)
    many = lines.attention(token)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)
        assert torch.equal(chunk.attention(queries, causal=True), whole)
        assert torch.equal(lines.attention(token), many)
    ex.synchronize(torch.cuda.current_stream())


def test_a_captured_chunk_outlives_other_calls(ex):
    """The same for a captured prompt chunk (split keys and the join)."""
    import torch
    cache = _filled(ex, 1, 1, 2000, 4, 64)
    q = _draw(2, 1, 40, 8, 64)
    out = torch.zeros_like(q)
    graph = _capture(lambda: cache.attention(q, out, causal=True))
    graph.replay()
    first = out.clone()
    step, step_out = _decoding_step(ex)
    step()
    want = step_out.clone()
    wide = _filled(ex, 7, 2, 5000, 8, 128)
    wide.attention(_draw(9, 2, 290, 16, 128))
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)
        step()
        assert torch.equal(step_out, want)


def test_launches_of_different_shares_alternate(ex):
    """Calls that cut the same workspace differently, one behind the other without a synchronisation."""
    import torch
    shapes = [(2, 1, 8, 4, 128, 9000), (1, 4, 8, 4, 64, 12000), (5, 1, 16, 8, 128, 3000), (40, 2, 8, 8, 64, 500),
              (1, 64, 8, 4, 128, 3000), (3, 17, 8, 4, 64, 2000)]
    caches, queries = [], []
    for i, (b, n, h, hk, d, keys) in enumerate(shapes):
        caches.append(_filled(ex, 10 * i, b, keys, hk, d, "e4m3" if i % 2 else "int8"))
        queries.append(_draw(10 * i + 2, b, n, h, d))
    want = []
    for c, q in zip(caches, queries):
        want.append(c.attention(q))
        ex.synchronize(torch.cuda.current_stream())
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    outs = [torch.empty_like(w) for w in want]
    for i in range(120):
        order = [(i * k + j) % len(shapes) for k in (1, 5) for j in range(len(shapes))]
        for j in order:
            caches[j].attention(queries[j], outs[j])
        for o, w in zip(outs, want):
            differ += (o.view(torch.int16) != w.view(torch.int16)).any()
    assert int(differ) == 0


def test_a_graph_outlives_larger_scratch(ex):
    """The context's scratch (normalised q, decoded weights) of a captured call, outgrown twice before the replay."""
    import torch
    cache = _filled(ex, 1, 1, 700, 8, 128)
    q, w = _draw(2, 1, 40, 8, 128), _draw(3, 128)
    out = torch.zeros_like(q)
    graph = _capture(lambda: cache.attention(q, out, qk_norm="rms", q_norm_weight=w))
    graph.replay()
    first = out.clone()
    plain = _draw(4, 1, 300, 16, 128)
    self_out = torch.zeros_like(plain)
    self_graph = _capture(lambda: ex.attention(plain, plain, plain, self_out, qk_norm="rms"))  # a larger scratch
    self_graph.replay()
    self_first = self_out.clone()
    big = _draw(5, 1, 3000, 8, 128)
    want = cache.attention(big, qk_norm="rms", q_norm_weight=w)                               # larger again
    taken = [torch.full((1 << 20,), 7.0, dtype=torch.float16, device="cuda") for _ in range(8)]
    for _ in range(3):
        out.zero_()
        self_out.zero_()
        graph.replay()
        self_graph.replay()
        assert torch.equal(out, first) and torch.equal(self_out, self_first)
        assert torch.equal(cache.attention(big, qk_norm="rms", q_norm_weight=w), want)
    assert all((t == 7).all() for t in taken)


def test_scratch_that_no_graph_holds_is_given_back(ex):
    """Eager calls of growing size keep one scratch buffer, not all of them: six sizes up to 96 MB, in 200 MB."""
    import torch
    torch.cuda.synchronize()
    qs = [torch.zeros((1, 4096 * n, 16, 128), dtype=torch.float16, device="cuda") for n in (1, 2, 3, 4, 5, 6)]
    k = torch.zeros((1, 64, 16, 128), dtype=torch.float16, device="cuda")
    out = torch.empty_like(qs[-1])
    ex.attention(qs[0], k, k, out[:, :4096], qk_norm="rms", qk_norm_targets="q")
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for n, q in enumerate(qs, 1):
        ex.attention(q, k, k, out[:, :4096 * n], qk_norm="rms", qk_norm_targets="q")
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] < 200 << 20


def test_a_timeout_is_cleared_on_the_callers_stream(ex):
    """A wait that runs out (1 ms, on a phase that nothing completes) on a non-blocking stream while the legacy stream
    is busy: it is reported and cleared without waiting for the other stream, and the split attention that follows
    at once has the right bits."""
    import torch

    from animaxs_b200 import AttentionTimeoutError
    step, out = _decoding_step(ex)
    step()
    want = out.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert ex._lib.animaxs_attn_selftest_wait_timeout(ex.handle, 1_000_000, side.cuda_stream) == 0
    with pytest.raises(AttentionTimeoutError):             # a kernel's first launch loads it, which waits for the device
        ex.synchronize(side)
    torch.cuda._sleep(1_000_000_000)                       # about half a second on the legacy stream
    busy = torch.cuda.Event()
    busy.record()
    with torch.cuda.stream(side):
        for _ in range(3):
            assert ex._lib.animaxs_attn_selftest_wait_timeout(ex.handle, 1_000_000, side.cuda_stream) == 0
            with pytest.raises(AttentionTimeoutError):
                ex.synchronize(side)
            for _ in range(20):
                step()
            ex.synchronize(side)                           # the status is clear again
            waited = busy.query()
            assert not waited, "the reset was not on the caller's stream"
    torch.cuda.synchronize()
    assert torch.equal(out, want)
