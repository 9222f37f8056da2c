"""GPU: the context's counters see attention over the 8-bit cache as they see other attention."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    from animaxs_b200 import AttentionExecutor
    e = AttentionExecutor(0)
    yield e
    e.close()


@pytest.mark.parametrize("batch,q_len,heads,keys", [(2, 1, 4, 300), (1, 130, 2, 64), (3, 300, 6, 2000), (1, 8, 2, 9000)])
def test_query_tiles_and_kernel_timing(ex, batch, q_len, heads, keys):
    """(head, 128-row tile) units, and one timed launch a call (the join of split keys within it)."""
    import torch

    from animaxs_b200 import QuantizedKVCache
    cache = QuantizedKVCache(ex, batch=batch, capacity=keys, kv_heads=2, head_dim=64)
    q = torch.zeros((batch, q_len, heads, 64), dtype=torch.float16, device="cuda")
    want = cache.attention(q)
    tiles = ex.attention_query_tiles
    ex.set_kernel_timing(True)
    try:
        for _ in range(3):
            out = cache.attention(q)
    finally:
        ex.set_kernel_timing(False)
    ex.synchronize(torch.cuda.current_stream())
    launches, total, most = ex.kernel_timing()
    assert launches == 3 and 0 < most <= total < 1000
    assert ex.attention_query_tiles - tiles == 3 * batch * heads * -(-q_len // 128)
    cache.attention(q)
    assert ex.kernel_timing()[0] == 0 and torch.equal(out, want)
