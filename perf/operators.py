"""Timing cases of the 8-bit K/V cache: writing it, reading it back, and attention over it.

The cache holds ``[batch][kv_heads][capacity][head_dim]`` codes (int8 or e4m3) for K and for V with one fp32
scale for each head and block of 64 tokens.  ``run`` computes a case in plain torch operations (``own`` false) or
through ``animaxs_b200.QuantizedKVCache`` (``own`` true).
"""

import math
import random

import torch

own = False

BLOCK = 64                                   # tokens that share a scale
TOP = {"int8": 127.0, "e4m3": 448.0}         # largest magnitude of a code
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------------------------------------- cases
def _write(name, batch, tokens, kv_heads, head_dim, capacity, start, fmt, ragged):
    return {"name": name, "op": "write", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
            "capacity": capacity, "start": start, "format": fmt, "ragged": ragged}


def _read(name, batch, tokens, kv_heads, head_dim, capacity, start, fmt, ragged):
    return {"name": name, "op": "read", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
            "capacity": capacity, "start": start, "format": fmt, "ragged": ragged}


def _attend(name, batch, q_len, kv_len, heads, kv_heads, head_dim, capacity, fmt, causal, ragged):
    return {"name": name, "op": "attend", "batch": batch, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "capacity": capacity, "format": fmt, "causal": causal,
            "ragged": ragged}


def listed():
    return [
        # One new token of each of 8 sequences, at ragged places in half-filled blocks: a decoding step's append.
        _write("write_token", 8, 1, 8, 128, 2048, 1300, "int8", True),
        # The DiT's cross K/V of one block for 8 prompts: 512 context tokens, 16 heads of 128, written once.
        _write("write_context", 8, 512, 16, 128, 512, 0, "int8", False),
        # Two long prompts of ragged lengths behind a cached prefix that ends inside a block.
        _write("write_long", 2, 16385, 8, 128, 16640, 37, "e4m3", True),
        # The same cross K/V read back as fp16 for a kernel that takes only that, prompts of ragged lengths.
        _read("read_context", 8, 512, 16, 128, 512, 0, "e4m3", True),
        # A long cached prompt read back (to move it to another format or device).
        _read("read_long", 1, 32741, 8, 128, 32768, 0, "int8", False),
        # One token on a prompt of the text encoder's size: 16 query heads on 8, 300 tokens; latency counts.
        _attend("token_prompt", 1, 1, 300, 16, 8, 128, 512, "int8", False, False),
        # A decoding step of a batch of 32 with ragged caches.
        _attend("token_batch", 32, 1, 4096, 16, 8, 128, 4096, "int8", False, True),
        # One token on one long cache: the work has to be split along the keys.
        _attend("token_long", 1, 1, 131071, 16, 8, 128, 131072, "e4m3", False, False),
        # Five new tokens at once on the adapter's heads of 64, causal among themselves.
        _attend("few_tokens", 4, 5, 1000, 16, 16, 64, 1024, "int8", True, True),
        # The DiT's cross attention of a 1024 x 1024 image: 4096 queries on 512 context tokens, 128 of them valid.
        _attend("cross_image", 1, 4096, 128, 16, 16, 128, 512, "int8", False, False),
        # The same for 8 images with prompts of ragged lengths.
        _attend("cross_batch", 8, 4096, 512, 16, 16, 128, 512, "int8", False, True),
        # A chunk of 512 prompt tokens on a cache of 8704, causal.
        _attend("prompt_chunk", 2, 512, 8704, 16, 8, 128, 8704, "e4m3", True, False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    fmt = rng.choice(["int8", "e4m3"])
    ragged = rng.random() < 0.5
    kind = rng.choice(["write", "read", "few", "few", "many", "many"])
    head_dim = rng.choice([128, 128, 64])
    kv_heads = rng.choice([1, 2, 8, 8, 16])
    if kind in ("write", "read"):
        batch = _log(rng, 1, 16)
        tokens = _log(rng, 1, 40_000_000 // (batch * kv_heads * head_dim * 4))
        tokens = min(tokens, 40_000)
        start = rng.choice([0, _log(rng, 1, 3000)])
        capacity = start + tokens + rng.choice([0, 1, 200])
        return (_write if kind == "write" else _read)("", batch, tokens, kv_heads, head_dim, capacity, start, fmt, ragged)
    group = rng.choice([1, 2, 2, 4, 7])
    heads = kv_heads * group
    if kind == "few":      # up to 16 rows for each key head, caches from one token to long ones
        q_len = rng.choice([1, 1, 1, max(1, 16 // group)])
        batch = _log(rng, 1, 48)
        kv_len = _log(rng, 1, min(131072, 130_000_000 // (batch * kv_heads * head_dim)))
        kv_len = max(kv_len, q_len)
    else:                  # images and prompt chunks
        batch = _log(rng, 1, 8)
        q_len = _log(rng, 17, min(4096, 500_000 // (batch * heads)))
        kv_len = _log(rng, 1, max(1, min(9000, 130_000_000 // (batch * heads * q_len))))
    causal = kv_len >= q_len and rng.random() < 0.5
    capacity = kv_len + rng.choice([0, 3, 64])
    return _attend("", batch, q_len, kv_len, heads, kv_heads, head_dim, capacity, fmt, causal, ragged)


def _lens(case, most):
    """Each sequence's count of tokens: ``most``, or ragged from a twentieth of it to all of it."""
    if not case["ragged"]:
        return [most] * case["batch"]
    rng = random.Random(1000 * case["batch"] + most)
    return [most if i == 0 else _log(rng, max(1, most // 20), most) for i in range(case["batch"])]


def _starts(case):
    """Where each sequence's new tokens go: ``start``, or ragged up to it."""
    if not case["ragged"]:
        return [case["start"]] * case["batch"]
    rng = random.Random(7 * case["batch"] + case["start"])
    return [rng.randint(0, case["start"]) for _ in range(case["batch"])]


# -------------------------------------------------------------------------------------------- inputs
def _keys(g, shape):
    """Keys as a normalising projection gives them: normal, with a few large channels."""
    x = torch.randn(shape, generator=g, device="cuda")
    x[..., 3::29] *= 4.0
    return x.half()


def _values(g, shape):
    return torch.randn(shape, generator=g, device="cuda").half()


def _encode(x, fmt):
    """Codes and scales of whole blocks of ``[batch, heads, capacity, dim]``."""
    b, h, t, d = x.shape
    pad = -t % BLOCK
    y = torch.nn.functional.pad(x.float(), (0, 0, 0, pad)).view(b, h, -1, BLOCK, d)
    scale = y.abs().amax((3, 4)) / TOP[fmt]
    y = (y / scale.clamp_min(1e-30)[..., None, None]).view(b, h, -1, d)[:, :, :t]
    codes = y.round().to(torch.int8) if fmt == "int8" else y.to(CODE[fmt])
    return codes.contiguous(), scale.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    fmt, b, h, d, cap = case["format"], case["batch"], case["kv_heads"], case["head_dim"], case["capacity"]
    state = {"case": case, "format": fmt}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for name, make in (("k", _keys), ("v", _values)):
        state[name + "_codes"], state[name + "_scale"] = _encode(make(g, (b, h, cap, d)), fmt)
    if case["op"] == "write":
        # [batch, tokens, heads, dim] slices of one projection's K|V rows.
        rows = torch.empty((b, case["tokens"], 2, h, d), dtype=torch.float16, device="cuda")
        rows[:, :, 0] = _keys(g, (b, case["tokens"], h, d))
        rows[:, :, 1] = _values(g, (b, case["tokens"], h, d))
        state["k"], state["v"] = rows[:, :, 0], rows[:, :, 1]
        state["starts"] = ints(_starts(case))
        state["counts"] = ints(_lens(case, case["tokens"]))
    elif case["op"] == "read":
        state["lens"] = ints([case["start"] + n for n in _lens(case, case["tokens"])])
    else:
        lens = ints(_lens(case, case["kv_len"]))
        state["lens"] = lens
        state["q"] = torch.randn((b, case["q_len"], case["heads"], d), generator=g, device="cuda").half()
        # What lies behind a sequence's last token is whatever the memory held: for e4m3 that may be NaN.
        if fmt == "e4m3":
            dead = torch.arange(cap, device="cuda")[None, :] >= lens[:, None]
            for name in ("k_codes", "v_codes"):
                state[name].view(torch.uint8).masked_fill_(dead[:, None, :, None], 0x7F)
    return state


# ------------------------------------------------------------------------------------- the framework
_executor = None


def _cache(state):
    """The program's cache object over its buffers, made once."""
    global _executor
    if "cache" not in state:
        import animaxs_b200
        if _executor is None:
            _executor = animaxs_b200.AttentionExecutor(0)
        state["cache"] = animaxs_b200.QuantizedKVCache.wrap(
            _executor, state["k_codes"], state["v_codes"], state["k_scale"], state["v_scale"])
    return state["cache"]


def _run_own(state):
    case, cache = state["case"], _cache(state)
    if case["op"] == "write":
        cache.write(state["k"], state["v"], starts=state["starts"], counts=state["counts"])
        return {"k_codes": cache.k_codes, "v_codes": cache.v_codes, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    if case["op"] == "read":
        k, v = cache.read(start=case["start"], tokens=case["tokens"], lens=state["lens"])
        return {"k": k, "v": v}
    return cache.attention(state["q"], lens=state["lens"], kv_len=case["kv_len"], causal=case["causal"])


# ---------------------------------------------------------------------------------------- plain forms
def _write_plain(state, x, codes, scale):
    case, top = state["case"], TOP[state["format"]]
    b, t, h, d = x.shape
    cap = codes.shape[2]
    start, count = state["starts"].long(), state["counts"].long()
    # The window of whole blocks that any sequence's new tokens can touch.
    width = ((t + BLOCK - 2) // BLOCK + 1) * BLOCK
    first = start // BLOCK * BLOCK
    pos = first[:, None] + torch.arange(width, device=x.device)             # [b, width] cache positions
    src = pos - start[:, None]                                              # index among the new tokens
    new = (src >= 0) & (src < count[:, None]) & (pos < cap)
    older = (src < 0) & (pos < cap)
    fresh = torch.gather(x.float(), 1, src.clamp(0, t - 1)[:, :, None, None].expand(-1, -1, h, d))
    fresh = torch.where(new[:, :, None, None], fresh, 0.0).transpose(1, 2)  # [b, h, width, d]
    blocks = lambda v: v.reshape(b, h, -1, BLOCK, d)                         # noqa: E731
    amax = blocks(torch.where(fresh.isfinite(), fresh.abs(), 0.0)).amax((3, 4))
    wrote = new.view(b, -1, BLOCK).any(2)                                   # blocks that get a token
    held = older.view(b, -1, BLOCK).any(2)                                  # blocks that keep older ones
    at = (pos[:, ::BLOCK] // BLOCK).clamp(max=scale.shape[2] - 1)[:, None, :].expand(-1, h, -1)
    before = torch.gather(scale, 2, at)
    s = torch.maximum(amax / top, torch.where(held[:, None], before, 0.0))
    s = torch.where(wrote[:, None], s, before)
    inverse = torch.where(s > 0, 1.0 / s, 0.0)
    whole = lambda v: v.round().clamp(-top, top) if state["format"] == "int8" else v.clamp(-top, top)  # noqa: E731
    index = pos.clamp(max=cap - 1)[:, None, :, None].expand(-1, h, -1, d)
    raw = codes.view(torch.int8)
    old = torch.gather(raw, 2, index)
    shrunk = blocks(old.view(codes.dtype).float()) * (before * inverse)[..., None, None]
    grown = (wrote & held)[:, None] & (s > before)
    quantised = whole(torch.nan_to_num(blocks(fresh), nan=0.0, posinf=math.inf, neginf=-math.inf)
                      * inverse[..., None, None])
    quantised = torch.nan_to_num(quantised, nan=0.0)
    new_b, old_b = new.view(b, 1, -1, BLOCK, 1), older.view(b, 1, -1, BLOCK, 1)
    value = torch.where(new_b, quantised.to(codes.dtype).view(torch.int8), blocks(old))
    value = torch.where(old_b & grown[..., None, None], whole(shrunk).to(codes.dtype).view(torch.int8), value)
    # A position past the capacity stands for the last one, value and all, so what is stored twice is equal.
    within = (pos.clamp(max=cap - 1) - first[:, None])[:, None, :, None].expand(-1, h, -1, d)
    raw.scatter_(2, index, torch.gather(value.reshape(b, h, width, d), 2, within))
    within = (pos[:, ::BLOCK] // BLOCK).clamp(max=scale.shape[2] - 1) - first[:, None] // BLOCK
    scale.scatter_(2, at, torch.gather(s, 2, within[:, None, :].expand(-1, h, -1)))


def _decoded(codes, scale):
    t = codes.shape[2]
    return codes.float() * scale.repeat_interleave(BLOCK, 2)[:, :, :t, None]


def _read_plain(state, codes, scale):
    case = state["case"]
    at = slice(case["start"], case["start"] + case["tokens"])
    x = _decoded(codes, scale)[:, :, at]
    pos = torch.arange(at.start, at.stop, device=codes.device)
    live = pos[None, :] < state["lens"][:, None]
    return torch.where(live[:, None, :, None], x, 0.0).half().transpose(1, 2).contiguous()


def _attend_plain(state):
    case = state["case"]
    n, group, i = case["kv_len"], case["heads"] // case["kv_heads"], case["q_len"]
    k = _decoded(state["k_codes"], state["k_scale"])[:, :, :n]
    v = _decoded(state["v_codes"], state["v_scale"])[:, :, :n]
    q = state["q"].float()
    b, _, h, d = q.shape
    pos = torch.arange(n, device=q.device)
    live = pos[None, :] < state["lens"][:, None]                            # [b, n]
    k = torch.where(live[:, None, :, None], k, 0.0)
    v = torch.where(live[:, None, :, None], v, 0.0)
    q = q.transpose(1, 2).reshape(b, case["kv_heads"], group * i, d)
    s = q @ k.transpose(2, 3) / math.sqrt(d)
    seen = live[:, None, None, :]
    if case["causal"]:
        last = state["lens"][:, None] - i + torch.arange(i, device=q.device)  # [b, i] own positions
        seen = seen & (pos <= last[:, :, None])[:, None]
    s = s.view(b, case["kv_heads"], group, i, n).masked_fill(~seen[:, :, None], -math.inf)
    top = s.amax(4, keepdim=True).clamp_min(-3e38)
    p = torch.exp(s - top)
    total = p.sum(4, keepdim=True)
    o = (p.view(b, case["kv_heads"], group * i, n) @ v).view(b, h, i, d)
    o = torch.where(total.view(b, h, i, 1) > 0, o / total.view(b, h, i, 1), 0.0)
    return o.transpose(1, 2).half().contiguous()


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "write":
        _write_plain(state, state["k"], state["k_codes"], state["k_scale"])
        _write_plain(state, state["v"], state["v_codes"], state["v_scale"])
        return {name: state[name] for name in ("k_codes", "v_codes", "k_scale", "v_scale")}
    if op == "read":
        return {"k": _read_plain(state, state["k_codes"], state["k_scale"]),
                "v": _read_plain(state, state["v_codes"], state["v_scale"])}
    return _attend_plain(state)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    h, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "write":
        n = sum(_lens(case, case["tokens"]))
        return {"bytes": 2 * n * h * d * 3 + 2 * 4 * h * (n // BLOCK + case["batch"]), "flops": 0}
    if case["op"] == "read":
        n = sum(_lens(case, case["tokens"]))
        return {"bytes": 2 * h * d * (n + 2 * case["batch"] * case["tokens"]) + 2 * 4 * h * (n // BLOCK), "flops": 0}
    lens, i = _lens(case, case["kv_len"]), case["q_len"]
    pairs = sum(sum(max(0, n - i + j + 1) for j in range(i)) if case["causal"] else n * i for n in lens)
    n = sum(lens)
    return {"bytes": 2 * n * h * d + 2 * 4 * h * (n // BLOCK + case["batch"]) + 4 * case["batch"] * i * case["heads"] * d,
            "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------------------------ in 64 bits
def _to_e4m3(x):
    """float64 values rounded to e4m3 (three bits of mantissa, least exponent -6), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_write(case, x, codes, scale, starts, counts):
    top, fmt = TOP[case["format"]], case["format"]
    values, scale = codes.double(), scale.double()
    rounded = _to_e4m3 if fmt == "e4m3" else torch.round
    for b in range(case["batch"]):
        p, n = starts[b], min(counts[b], case["capacity"] - starts[b])
        if n <= 0:
            continue
        edge = p // BLOCK * BLOCK
        fresh = x[b, :n].double().transpose(0, 1)                           # [h, n, d]
        held = (values[b, :, edge:p] * scale[b, :, p // BLOCK, None, None]) if p > edge else None
        whole = torch.zeros((fresh.shape[0], (-(-(p + n) // BLOCK)) * BLOCK - edge, fresh.shape[2]),
                            dtype=torch.float64, device=x.device)
        whole[:, p - edge:p - edge + n] = fresh
        s = whole.view(fresh.shape[0], -1, BLOCK, fresh.shape[2]).abs().amax((2, 3)) / top
        if held is not None:
            before = scale[b, :, p // BLOCK].clone()
            s[:, 0] = torch.maximum(s[:, 0], before)
            grown = s[:, 0] > before
            values[b, grown, edge:p] = rounded(held[grown] / s[grown, 0, None, None])
        first = p // BLOCK
        scale[b, :, first:first + s.shape[1]] = s
        wide = s.repeat_interleave(BLOCK, 1)[:, p - edge:p - edge + n, None]
        values[b, :, p:p + n] = rounded(fresh / wide.clamp_min(1e-300))
    # int8 codes are whole numbers whose ties are decided in 32 bits: they have no value in 64.
    return (values if fmt == "e4m3" else None), scale


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "write":
        starts, counts = _starts(case), _lens(case, case["tokens"])
        k = _exact_write(case, state["k"], state["k_codes"], state["k_scale"], starts, counts)
        v = _exact_write(case, state["v"], state["v_codes"], state["v_scale"], starts, counts)
        return {"k_codes": k[0], "v_codes": v[0], "k_scale": k[1], "v_scale": v[1]}
    blocks = torch.arange(case["capacity"], device="cuda") // BLOCK
    if case["op"] == "read":
        out = {}
        for name in ("k", "v"):
            x = state[name + "_codes"].double() * state[name + "_scale"].double()[:, :, blocks, None]
            x = x[:, :, case["start"]:case["start"] + case["tokens"]].transpose(1, 2).contiguous()
            for b, n in enumerate(_lens(case, case["tokens"])):
                x[b, n:] = 0
            out[name] = x
        return out
    group, i, d = case["heads"] // case["kv_heads"], case["q_len"], case["head_dim"]
    out = torch.zeros((case["batch"], i, case["heads"], d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case, case["kv_len"])):
        later = torch.arange(n, device="cuda")[None, :] > (n - i + torch.arange(i, device="cuda"))[:, None]
        for h in range(case["kv_heads"]):
            k = state["k_codes"][b, h, :n].double() * state["k_scale"][b, h].double()[blocks[:n], None]
            v = state["v_codes"][b, h, :n].double() * state["v_scale"][b, h].double()[blocks[:n], None]
            for a in range(h * group, (h + 1) * group):
                s = state["q"][b, :, a].double() @ k.t() * d ** -0.5
                if case["causal"]:
                    s[later] = -math.inf
                out[b, :, a] = torch.nan_to_num(torch.softmax(s, 1)) @ v
    return out
