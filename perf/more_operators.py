"""Timed and checked cases of the cache held in 4 bits: writing it, reading it back, and attention
over it.

`own` False computes each operator from elementary torch operations in 32 bits (64 where a value
next to a border of two codes needs them); `own` True calls the package's entry points
(kv_quantize, kv_dequantize, quantized_attention).  Shapes: queries [rows, tokens, heads,
head_dim]; new keys and values [rows, kv_heads, tokens, head_dim]; one layer's cache uint8 [rows,
kv_heads, capacity, record].

A record holds one slot of one head: the codes c of the dimensions (4 bits each, dimensions rounded
up to a multiple of 32), then four pairs of float16, scale and middle of a group of dimensions (32
of them; 16 where there are at most 64): a value stands for mid + scale (c - 8).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
CLAMP = 32768.0  # finite values beyond count as this

# The largest listed case (the long chunk) bounds the drawn ones: heads x queries x slots of its score
# matrix, the values of any cache, and those of a prompt that is written.
MOST_SCORES = 36 * 2048 * 16384
MOST_VALUES = 64 * 4 * 8192 * 128
MOST_WRITTEN = 8 * 4 * 8192 * 128


def _write(name, dtype, rows, tokens, kv_heads, head_dim, capacity, fused=False, ragged=True):
    c = {"op": "write", "dtype": dtype, "rows": rows, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
         "capacity": capacity, "fused": fused, "ragged": ragged}
    return {"name": name, **c} if name else c


def _read(name, dtype, rows, tokens, kv_heads, head_dim, capacity):
    c = {"op": "read", "dtype": dtype, "rows": rows, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
         "capacity": capacity}
    return {"name": name, **c} if name else c


def _attend(name, dtype, rows, tokens, heads, kv_heads, head_dim, capacity, window=0, sinks=0, ragged=True):
    c = {"op": "attend", "dtype": dtype, "rows": rows, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "capacity": capacity, "window": window, "sinks": sinks, "ragged": ragged}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One token of two beams of the 1B decoder goes into the cache: latency is all.
        _write("write token 1b beams", "f16", 2, 1, 1, 128, 1024),
        # A long prompt of the 8B decoder, taken in place from the fused projection (36 + 4 + 4 heads).
        _write("write prompt 8b", "bf16", 1, 8192, 4, 128, 8192, fused=True, ragged=False),
        # Prompts of an image's tokens in full precision, ragged, small heads.
        _write("write prompts f32", "f32", 4, 577, 8, 64, 1001),
        # The cache of two beams, whole and small.
        _read("read cache 1b", "f16", 2, 1024, 1, 128, 1024),
        # The last window of a few sequences, for a kernel that wants 16-bit values.
        _read("read window 8b", "bf16", 8, 4096, 4, 128, 8192),
        # Two beams of the 1B decoder (16 heads, one key/value head), one token: latency again.
        _attend("token 1b beams", "f16", 2, 1, 16, 1, 128, 1024, 512, 4),
        # A few long sequences of the 8B decoder (36 heads over 4), one token each.
        _attend("token 8b long", "bf16", 8, 1, 36, 4, 128, 16384),
        # A serving batch of the same decoder with ragged lengths and its window: the cache's bytes count.
        _attend("token batch 8b", "bf16", 64, 1, 36, 4, 128, 8192, 4096, 4),
        # Full precision, as the 1B decoder runs without half types.
        _attend("token f32", "f32", 8, 1, 16, 1, 128, 2001),
        # Five drafted tokens of several sequences are checked at once.
        _attend("draft 8b", "bf16", 16, 5, 36, 4, 128, 4097, 4096, 4),
        # A chunk of a prompt against a filled cache, small heads.
        _attend("chunk d64", "f16", 4, 100, 32, 8, 64, 6000, 2048, 64),
        # A long chunk against a long cache: the largest case.
        _attend("chunk long 8b", "bf16", 1, 2048, 36, 4, 128, 16384, ragged=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8, 9, 16] if kv > 1 else [1, 4, 8, 12, 16])
    return kv * group, kv


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["write", "write token", "read", "token", "token", "token", "draft", "chunk", "chunk"])
    dtype = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 80, 128, 128, 128])
    while True:
        heads, kv = _heads(rng)
        if kind == "write":
            rows, tokens = _log(rng, 1, 8), _log(rng, 16, 8192)
            if rows * tokens * kv * dim <= MOST_WRITTEN:
                return _write(None, dtype, rows, tokens, kv, dim, tokens + rng.choice([0, _log(rng, 1, 1024)]),
                              fused=rng.random() < 0.5)
        elif kind == "write token":
            rows, tokens, capacity = _log(rng, 1, 64), _log(rng, 1, 8), _log(rng, 64, 8192)
            if rows * kv * capacity * dim <= MOST_VALUES:
                return _write(None, dtype, rows, tokens, kv, dim, capacity)
        elif kind == "read":
            rows, capacity = _log(rng, 1, 64), _log(rng, 64, 8192)
            tokens = rng.choice([capacity, _log(rng, 1, capacity)])
            if rows * kv * tokens * dim <= MOST_WRITTEN and rows * kv * capacity * dim <= MOST_VALUES:
                return _read(None, dtype, rows, tokens, kv, dim, capacity)
        else:
            rows = _log(rng, 1, 64 if kind != "chunk" else 8)
            capacity = _log(rng, 64, 16384)
            tokens = {"token": 1, "draft": _log(rng, 2, 8), "chunk": _log(rng, 9, min(2048, capacity))}[kind]
            window = rng.choice([0, 0, _log(rng, 16, 4096)])
            scores = rows * heads * tokens * capacity * (8 if dtype == "f32" else 1)
            if rows * kv * capacity * dim <= MOST_VALUES and scores <= MOST_SCORES // 2:
                return _attend(None, dtype, rows, tokens, heads, kv, dim, capacity, window,
                               rng.choice([0, 1, 4, 64]) if window else 0)


def _padded(dim):
    return (dim + 31) // 32 * 32


def _group(dim):
    return 32 if _padded(dim) >= 96 else 16


def _record(dim):
    return _padded(dim) // 2 + 16


def _spread(low, high, n, g):
    """n lengths from low to high, evenly spread, in an order made from the generator."""
    v = torch.linspace(low, high, n, dtype=torch.float64).round().to(torch.int32)
    return v[torch.randperm(n, generator=g)].cuda()


def _shortest(case):
    """Rows hold from half the capacity up to all of it; prompts that are written may be shorter than the
    longest of them (their first places are padding)."""
    c, n = case["capacity"], case["tokens"]
    if not case.get("ragged", True):
        return c
    return max(1, (n + 1) // 2) if case["op"] == "write" and n > 8 else max(n, (c + 1) // 2)


def prepare(case, seed):
    g, h = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    R, n, K, C, D = (case[k] for k in ("rows", "tokens", "kv_heads", "capacity", "head_dim"))
    s = dict(case)
    short = _shortest(case)
    s["lengths"] = _spread(short, C, R, h) if short < C else None
    # Keys lean to a direction of their own in each head, values do not.
    lean = torch.randn((K, 1, D), generator=g, device="cuda")

    def normal(slots, shift):
        return torch.randn((R, K, slots, D), generator=g, device="cuda") + shift

    if case["op"] == "write":
        k, v = normal(n, lean), normal(n, 0.0)
        if case["fused"]:  # a projection of queries, keys and values together: 9 queries a head
            x = torch.zeros((R, n, 11 * K * D), device="cuda", dtype=dtype)
            x[:, :, 9 * K * D:10 * K * D] = k.transpose(1, 2).reshape(R, n, K * D)
            x[:, :, 10 * K * D:] = v.transpose(1, 2).reshape(R, n, K * D)
            s["keys"] = x[:, :, 9 * K * D:10 * K * D].unflatten(2, (K, D)).transpose(1, 2)
            s["values"] = x[:, :, 10 * K * D:].unflatten(2, (K, D)).transpose(1, 2)
        else:
            s["keys"], s["values"] = k.to(dtype), v.to(dtype)
        s["cache_keys"] = torch.zeros((R, K, C, _record(D)), device="cuda", dtype=torch.uint8)
        s["cache_values"] = torch.zeros_like(s["cache_keys"])
        return s
    s["cache_keys"] = torch.empty((R, K, C, _record(D)), device="cuda", dtype=torch.uint8)
    s["cache_values"] = torch.empty_like(s["cache_keys"])
    step = max(1, (1 << 26) // (K * C * D))  # rows at a time
    for name, shift in (("cache_keys", lean), ("cache_values", 0.0)):
        for r in range(0, R, step):
            x = torch.randn((min(step, R - r), K, C, D), generator=g, device="cuda") + shift
            s[name][r:r + step] = _pack(x)
    if case["op"] == "attend":
        q = torch.randn((R, n, K, case["heads"] // K, D), generator=g, device="cuda") + 0.5 * lean.view(K, 1, D)
        s["q"] = q.flatten(2, 3).to(dtype)
    return s


def _package():
    from __graft_entry__ import load_package
    return load_package()


_sv = []


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[state["op"]](state)


def _own(s):
    if not _sv:
        _sv.append(_package())
    sv = _sv[0]
    if s["op"] == "attend":
        return {"out": sv.quantized_attention(s["q"], s["cache_keys"], s["cache_values"], s["lengths"],
                                              window=s["window"], sinks=s["sinks"])}
    if s["op"] == "write":
        sv.kv_quantize(s["keys"], s["values"], s["cache_keys"], s["cache_values"], s["lengths"])
    # What the records stand for (of a write: of those it wrote).
    keys, values = sv.kv_dequantize(s["cache_keys"], s["cache_values"], s["head_dim"], s["lengths"],
                                    tokens=s["tokens"], dtype=DTYPES[s["dtype"]])
    return {"keys": keys, "values": values}


def _half(x):
    """float64 to float16, rounded once: through a float32 whose last bit remembers what it lost."""
    f = x.float()
    bits = torch.where(f.double() != x, (f.view(torch.int32) - (f.double().abs() > x.abs()).int()) | 1,
                       f.view(torch.int32))
    return bits.view(torch.float32).half()


def _pack(x):
    """Values [..., head_dim] as records uint8 [..., record]."""
    D = x.shape[-1]
    P, G = _padded(D), _group(D)
    x = x.float()
    ok = torch.isfinite(x)
    x = x.clamp(-CLAMP, CLAMP)
    pad = torch.nn.functional.pad
    low = pad(x, (0, P - D), value=math.inf).unflatten(-1, (P // G, G)).amin(-1)
    high = pad(x, (0, P - D), value=-math.inf).unflatten(-1, (P // G, G)).amax(-1)
    scale = _half((high.double() - low.double()) / 15)
    mid = _half(low.double() + 8 * scale.double())
    bad = ~pad(ok, (0, P - D), value=True).unflatten(-1, (P // G, G)).all(-1)
    scale, mid = scale.masked_fill(bad, math.nan), mid.masked_fill(bad, math.nan)
    m, s = mid.repeat_interleave(G, -1)[..., :D], scale.repeat_interleave(G, -1)[..., :D]
    # The quotient in 64 bits: ties between two codes go to the even one.
    c = torch.round((x.double() - m.double()) / torch.where(s == 0, 1.0, s.double())).float() * (s != 0) + 8
    c = torch.where(torch.isnan(c), 0.0, c).clamp(0, 15).to(torch.int32)
    # Word t P/32 + i: of the 32 dimensions of block i those at 4 t + 2 a + b (+ 16 e) in nibble 4 b + 2 e + a.
    c = pad(c, (0, P - D)).unflatten(-1, (P // 32, 2, 4, 2, 2)).movedim(-3, -5)  # [t, i, e, a, b]
    e = torch.arange(2, device=x.device)
    shift = 4 * (4 * e + 2 * e.view(2, 1, 1) + e.view(2, 1))
    low16 = (c[..., 0] << shift[..., 0]).sum((-1, -2)).to(torch.int32)
    high16 = (c[..., 1] << (shift[..., 1] - 16)).sum((-1, -2)).to(torch.int32)
    words = torch.stack([low16, high16], -1).flatten(-3)  # 16-bit halves, [t, i, half]
    codes = torch.stack([words & 255, words >> 8], -1).flatten(-2).to(torch.uint8)
    both = torch.stack([scale, mid], -1).flatten(-2)
    both = pad(both, (0, 8 - both.shape[-1])).contiguous().view(torch.uint8)
    return torch.cat([codes, both], -1)


def _unpack(records, D):
    """What records uint8 [..., record] stand for, float32 [..., head_dim]."""
    P, G = _padded(D), _group(D)
    b = records[..., :P // 2].unflatten(-1, (4, P // 32, 4))  # [t, i, byte]
    nibbles = torch.stack([b & 15, b >> 4], -1).flatten(-2)   # [t, i, nibble 4 b + 2 e + a]
    c = nibbles.unflatten(-1, (2, 2, 2)).movedim(-5, -3)      # [i, b, t, e, a] of [t, i, b, e, a]
    c = c.movedim(-2, -4).movedim(-3, -1)                     # [i, e, t, a, b]
    c = c.flatten(-5).float() - 8
    both = records[..., P // 2:].contiguous().view(torch.float16).unflatten(-1, (4, 2))[..., :P // G, :].float()
    x = both[..., 1].repeat_interleave(G, -1) + both[..., 0].repeat_interleave(G, -1) * c
    return x[..., :D]


def _newest(s):
    """The slots of the newest tokens, [rows, tokens], and which of them there are."""
    n, C, R = s["tokens"], s["capacity"], s["rows"]
    i = torch.arange(n, device=s["cache_keys"].device)
    at = i.expand(R, n) + (C - n) if s["lengths"] is None else s["lengths"][:, None].long() - n + i
    return at, at >= 0


def _plain_write(s):
    at, there = _newest(s)
    r, i = there.nonzero(as_tuple=True)
    for new, cache in (("keys", "cache_keys"), ("values", "cache_values")):
        s[cache][r, :, at[r, i]] = _pack(s[new])[r, :, i]
    return _plain_read(s)


def _plain_read(s):
    at, there = _newest(s)
    R, n, K, D = s["rows"], s["tokens"], s["kv_heads"], s["head_dim"]
    index = at.clamp_min(0)[:, None, :, None].expand(R, K, n, _record(D))
    see = there[:, None, :, None]
    return {name: torch.where(see, _unpack(s["cache_" + name].gather(2, index), D), 0.0).to(DTYPES[s["dtype"]])
            for name in ("keys", "values")}


def _plain_attend(s):
    q = s["q"].float()
    R, n, H, D = q.shape
    K, C = s["kv_heads"], s["capacity"]
    x = q.view(R, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(R, K, H // K * n, D)
    keys = _unpack(s["cache_keys"], D)
    scores = (torch.matmul(x, keys.transpose(2, 3)) * D ** -0.5).view(R, K, H // K, n, C)
    del keys
    slot = torch.arange(C, device=q.device)
    at = _newest(s)[0][:, None, None, :, None]
    see = slot <= at
    if s["window"]:
        see = see & ((slot > at - s["window"]) | (slot < s["sinks"]))
    scores = torch.where(see, scores, -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    scores = (scores / scores.sum(-1, keepdim=True)).view(R, K, H // K * n, C)
    out = torch.matmul(scores, _unpack(s["cache_values"], D)).view(R, K, H // K, n, D)
    return {"out": out.permute(0, 3, 1, 2, 4).reshape(R, n, H, D).to(s["q"].dtype)}


def work(case):
    e, D, R, n, K, C = BYTES[case["dtype"]], *(case[k] for k in ("head_dim", "rows", "tokens", "kv_heads", "capacity"))
    lengths = torch.linspace(_shortest(case), C, R, dtype=torch.float64).round()
    if case["op"] != "attend":
        slots = float(lengths.clamp(max=n).sum())
        values = 2 * K * D * e * (R * n + (slots if case["op"] == "write" else 0))
        return {"bytes": values + 2 * K * _record(D) * slots, "flops": 2 * K * D * slots * (8 if case["op"] == "write" else 2)}
    H, w, k = case["heads"], case["window"] or C, torch.tensor(float(case["sinks"]))
    at = lengths[:, None] - n + torch.arange(n)
    low = (at - w + 1).clamp(min=0)
    pairs = float((at + 1 - low + torch.minimum(low, k)).sum())
    slots = float((at[:, -1] + 1 - low[:, 0] + torch.minimum(low[:, 0], k)).sum())
    return {"bytes": R * n * H * D * e * 2 + 2 * K * _record(D) * slots, "flops": 4 * D * H * pairs}


def _stands_for(records, D):
    """What records (numpy, [slots, record]) stand for in 64 bits: one dimension at a time, from the format."""
    P, G = _padded(D), _group(D)
    words = np.ascontiguousarray(records[:, :P // 2]).view("<u4")
    both = np.ascontiguousarray(records[:, P // 2:]).view("<f2").astype(np.float64)
    x = np.empty((len(records), D))
    for d in range(D):
        i, y = divmod(d, 32)
        e, t, a, b = y >> 4, y >> 2 & 3, y >> 1 & 1, y & 1
        c = words[:, t * (P // 32) + i] >> np.uint32(4 * (4 * b + 2 * e + a)) & np.uint32(15)
        x[:, d] = both[:, 2 * (d // G) + 1] + both[:, 2 * (d // G)] * (c.astype(np.float64) - 8)
    return x


def _after_writing(x, D):
    """What values [slots, head_dim] (numpy, 64 bits) are once they have been held in 4 bits."""
    G, out = _group(D), np.empty_like(x)
    for d in range(0, D, G):
        y = np.clip(x[:, d:d + G], -CLAMP, CLAMP)
        low = y.min(1, keepdims=True)
        scale = ((y.max(1, keepdims=True) - low) / 15).astype(np.float16).astype(np.float64)
        mid = (low + 8 * scale).astype(np.float16).astype(np.float64)
        c = np.rint(np.divide(y - mid, scale, out=np.zeros_like(y), where=scale != 0))
        out[:, d:d + G] = mid + scale * np.clip(c, -8, 7)
    return out


def exact(case, seed):
    """The operators' definitions in 64 bits, one row and key/value head at a time."""
    s = prepare(case, seed)
    R, n, K, C, D = (case[k] for k in ("rows", "tokens", "kv_heads", "capacity", "head_dim"))
    ends = [C] * R if s["lengths"] is None else s["lengths"].tolist()
    if case["op"] != "attend":
        found = {}
        for name in ("keys", "values"):
            out = np.zeros((R, K, n, D))
            for r in range(R):
                for h in range(K):
                    m = min(n, ends[r])  # the newest m places hold tokens
                    if case["op"] == "write":
                        out[r, h, n - m:] = _after_writing(s[name][r, h, n - m:].double().cpu().numpy(), D)
                    else:
                        out[r, h, n - m:] = _stands_for(s["cache_" + name][r, h, ends[r] - m:ends[r]].cpu().numpy(), D)
            found[name] = torch.from_numpy(out)
        return found
    q, group = s["q"].double(), case["heads"] // K
    out = torch.zeros_like(q)
    for r in range(R):
        first = max(0, ends[r] - n - case["window"] + 1) if case["window"] and not case["sinks"] else 0
        j = torch.arange(first, ends[r], device=q.device)
        i = torch.arange(ends[r] - n, ends[r], device=q.device)[:, None]
        hidden = j > i
        if case["window"]:
            hidden |= (j <= i - case["window"]) & (j >= case["sinks"])
        for h in range(K):
            keys, values = (torch.from_numpy(_stands_for(s[x][r, h, first:ends[r]].cpu().numpy(), D)).cuda()
                            for x in ("cache_keys", "cache_values"))
            for g in range(h * group, (h + 1) * group):
                z = (q[r, :, g] @ keys.T).div_(math.sqrt(D)).masked_fill_(hidden, -math.inf)
                out[r, :, g] = torch.softmax(z, -1) @ values
    return {"out": out}
