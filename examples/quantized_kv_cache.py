"""The 8-bit K/V cache in two uses: ``python examples/quantized_kv_cache.py`` on a B200.

* DiT cross-attention: a block's K (RMS-normalised) and V over the adapter context are written once per generation
  and read by every Euler step, from codes instead of fp16.
* Decoding with the text encoder's heads (16 query and 8 key/value heads of 128): prompts of different lengths are written in chunks
  and attended causally; then every step appends one token to each sequence and attends to all of its cache, replayed
  from one CUDA graph, since positions and lengths are device tensors.

Each part returns (and prints) its largest difference from the fp16 path's output and from the written values."""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import animaxs_b200 as ax  # noqa: E402


def cross_attention(ex, *, blocks=4, steps=2, images=1, tokens=4096, context=512, heads=16, format="int8", seed=0):
    """``blocks`` DiT blocks over ``steps`` Euler steps with the context's K/V in fp16 and in 8 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: torch.randn(shape, generator=g, device="cuda").half()
    fp16 = ax.CrossKVCache(ex, blocks=blocks, batch=images, tokens=context, kv_heads=heads)
    codes = []
    for b in range(blocks):  # once per generation
        fp16.fill(b, draw(images, context, heads, 128), draw(images, context, heads, 128))  # K normalised here
        c = ax.QuantizedKVCache(ex, batch=images, capacity=context, kv_heads=heads, format=format)
        c.write(fp16.k(b), fp16.v(b))
        codes.append(c)
    worst = 0.0
    for _ in range(steps):
        for b in range(blocks):
            q = draw(images, tokens, heads, 128)
            want = ex.attention(q, fp16.k(b), fp16.v(b), qk_norm="rms", qk_norm_targets="q")
            got = codes[b].attention(q, qk_norm="rms")
            worst = max(worst, (got.float() - want.float()).abs().max().item())
    ex.synchronize()
    held = sum(c.nbytes for c in codes)
    k, _ = codes[0].read()
    stored = (k.float() - fp16.k(0).float()).abs().max().item()
    result = {"output_difference": worst, "value_difference": stored, "bytes": held,
              "fp16_bytes": blocks * fp16.block_stride}
    fp16.close()
    return result


def decode(ex, *, prompts=(300, 129, 1, 64), steps=32, chunk=128, heads=16, kv_heads=8, format="int8", seed=1):
    """Prompts in chunks, then ``steps`` tokens for all sequences; compared with one fp16 causal call over everything."""
    dim, batch, total = 128, len(prompts), max(prompts) + steps
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda h: torch.randn((batch, total, h, dim), generator=g, device="cuda").half()
    rope = torch.from_numpy(ax.qwen_rope(total)).cuda().view(total, -1)

    def rotate(x, positions):
        """Per-head RMSNorm and RoPE of ``x`` [n, h, dim] at ``positions`` [n], as the model does before the cache."""
        x, y = x.contiguous(), torch.empty_like(x)
        ex.rms_rope_split_half(torch.cuda.current_stream(), x, y, None, rope.index_select(0, positions),
                               tokens=x.shape[0], heads=x.shape[1], head_dim=dim)
        return y

    every = torch.arange(total, device="cuda").repeat(batch)
    q, k = (rotate(x.view(-1, x.shape[2], dim), every).view(x.shape) for x in (draw(heads), draw(kv_heads)))
    v = draw(kv_heads)

    cache = ax.QuantizedKVCache(ex, batch=batch, capacity=total, kv_heads=kv_heads, format=format)
    got = torch.zeros_like(q)
    first = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    for lo in range(0, max(prompts), chunk):  # prompts: ``counts`` cuts the shorter ones' last chunk
        hi = min(lo + chunk, max(prompts))
        starts = torch.full_like(first, lo)
        cache.write(k[:, lo:hi], v[:, lo:hi], starts=starts, counts=(first - lo).clamp(0, hi - lo))
        # A shorter prompt's queries past its end see positions that hold zeros so far; their rows are not used.
        got[:, lo:hi] = cache.attention(q[:, lo:hi], lens=starts + (hi - lo), kv_len=hi, causal=True)

    lens = first.clone()
    row = torch.arange(batch, device="cuda")
    k_t, v_t, q_t, o_t = (torch.empty((batch, 1, h, dim), dtype=torch.float16, device="cuda")
                          for h in (kv_heads, kv_heads, heads, heads))

    def step():
        at = lens.long()  # each sequence's next position
        q_t.copy_(q[row, at].unsqueeze(1))
        k_t.copy_(k[row, at].unsqueeze(1))
        v_t.copy_(v[row, at].unsqueeze(1))
        cache.write(k_t, v_t, starts=lens)
        lens.add_(1)
        cache.attention(q_t, o_t, lens=lens)
        got[row, at] = o_t.squeeze(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # the first call sizes the context's workspace, which a capture may not
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(steps - 1):
        graph.replay()
    ex.synchronize()

    used = torch.arange(total, device="cuda")[None, :] < lens[:, None]
    want = ex.attention(q, k, v, causal=True)
    k_read, _ = cache.read(lens=lens)
    return {"output_difference": (got.float() - want.float())[used].abs().max().item(),
            "value_difference": (k_read.float() - k.float())[used].abs().max().item(),
            "lengths": lens.tolist(), "bytes": cache.nbytes, "fp16_bytes": 2 * k.numel() * 2}


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--format", choices=("int8", "e4m3"), default="int8")
    args = parser.parse_args()
    ex = ax.AttentionExecutor(0)
    for name, part in (("cross-attention", cross_attention), ("decoding", decode)):
        print(name, args.format, part(ex, format=args.format))
    ex.close()


if __name__ == "__main__":
    main()
