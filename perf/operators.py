"""Timed and checked cases of the cache operators: attention with a sliding window and
sinks, attention over a shared prefix, and eviction by accumulated attention weight.

`own` False computes each operator from elementary torch operations in 32 bits;
`own` True calls the package's entry points (window_attention, prefix_attention,
kv_evict).  Shapes: queries [rows, tokens, heads, head_dim]; one layer's cache
[rows, kv_heads, capacity, head_dim]; a whole cache [layers, rows, kv_heads,
capacity, head_dim].
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}

# The largest listed case (the long prompt) bounds the drawn ones: heads x queries x
# slots of its score matrix, and the bytes of any cache.
MOST_SCORES = 36 * 8192 * 8192
MOST_CACHE = 1 << 30


def _window(name, dtype, rows, tokens, heads, kv_heads, head_dim, capacity, window, sinks, ragged=True, fused=False,
            weigh=False):
    c = {"op": "window", "dtype": dtype, "rows": rows, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "capacity": capacity, "window": window, "sinks": sinks, "ragged": ragged,
         "fused": fused, "weigh": weigh}
    return {"name": name, **c} if name else c


def _prefix(name, dtype, rows, tokens, heads, kv_heads, head_dim, prefix, capacity):
    c = {"op": "prefix", "dtype": dtype, "rows": rows, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "prefix": prefix, "capacity": capacity}
    return {"name": name, **c} if name else c


def _evict(name, dtype, layers, rows, kv_heads, head_dim, capacity, shortest, budget, sinks, recent):
    c = {"op": "evict", "dtype": dtype, "layers": layers, "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim,
         "capacity": capacity, "shortest": shortest, "budget": budget, "sinks": sinks, "recent": recent}
    return {"name": name, **c} if name else c


def listed():
    return [
        # Two beams of the 1B decoder (16 heads, one key/value head), one token: latency is all.
        _window("window token 1b beams", "f16", 2, 1, 16, 1, 128, 1024, 512, 4),
        # A few sequences of the 8B decoder (36 heads over 4, window 4096), one token each.
        _window("window token 8b", "bf16", 8, 1, 36, 4, 128, 8192, 4096, 4),
        # A serving batch of the same decoder with ragged lengths: the cache's bytes count.
        _window("window token batch", "bf16", 64, 1, 36, 4, 128, 8192, 4096, 4),
        # Prompts of an image's 577 tokens, keys and values read in place from the fused projection.
        _window("window prompt fused", "f16", 3, 577, 16, 1, 128, 577, 256, 1, ragged=True, fused=True),
        # A whole long prompt of the 8B decoder: the largest case.
        _window("window prompt long", "bf16", 1, 8192, 36, 4, 128, 8192, 4096, 4, ragged=False),
        # A chunk of a prompt against a filled cache, small heads.
        _window("window chunk d64", "bf16", 4, 100, 32, 8, 64, 6000, 2048, 64),
        # Full precision, as the 1B decoder runs without half types.
        _window("window prompt f32", "f32", 2, 333, 16, 1, 128, 1001, 512, 4),
        # Eight beams of the 1B decoder behind one image's prefix.
        _prefix("prefix beams 1b", "f16", 8, 1, 16, 1, 128, 1025, 512),
        # A serving batch behind one long system prompt, 8B heads.
        _prefix("prefix batch 8b", "bf16", 64, 1, 36, 4, 128, 8192, 1024),
        # One token's attention that also accumulates each slot's weight.
        _window("weights token 8b", "bf16", 8, 1, 36, 4, 128, 4097, 0, 0, weigh=True),
        # Every token of a full cache evicts one slot in each layer, row and head.
        _evict("evict step 8b", "bf16", 32, 8, 4, 128, 2304, 2049, 2048, 4, 256),
        # After a prompt: the 1B decoder's cache cut down to its budget.
        _evict("evict prompt 1b", "f16", 24, 2, 1, 128, 8192, 5000, 2048, 4, 512),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8, 9, 16] if kv > 1 else [1, 4, 8, 12, 16])
    return kv * group, kv


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["token", "token", "prompt", "prompt", "prefix", "prefix", "weights", "step", "prompt_evict"])
    dtype = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 80, 128, 128, 128])
    while True:
        heads, kv = _heads(rng)
        rows = _log(rng, 1, 64)
        capacity = _log(rng, 64, 8192)
        cache = 2 * rows * kv * capacity * dim * BYTES[dtype]
        if kind in ("token", "weights"):
            tokens = 1 if kind == "token" else rng.choice([1, 1, 1, _log(rng, 2, 256)])
            window = rng.choice([0, _log(rng, 16, 4096), _log(rng, 16, 4096)]) if kind == "token" else 0
            if tokens <= capacity and cache <= MOST_CACHE and rows * heads * tokens * capacity <= MOST_SCORES // 8:
                return _window(None, dtype, rows, tokens, heads, kv, dim, capacity, window,
                               rng.choice([0, 1, 4, 64]) if window else 0, weigh=kind == "weights")
        elif kind == "prompt":
            rows = _log(rng, 1, 8)
            tokens = _log(rng, 2, capacity)
            fused = rng.random() < 0.4
            scores = rows * heads * tokens * (tokens if fused else capacity)
            if scores * (4 if dtype == "f32" else 1) <= MOST_SCORES // 2:
                return _window(None, dtype, rows, tokens, heads, kv, dim, tokens if fused else capacity,
                               _log(rng, 16, 4096), rng.choice([0, 1, 4, 64]), fused=fused)
        elif kind == "prefix":
            prefix = _log(rng, 16, 8192)
            capacity = _log(rng, 8, 1024)
            tokens = rng.choice([1, 1, 1, _log(rng, 2, 16)])
            cache = 2 * (rows * capacity + prefix) * kv * dim * BYTES[dtype]
            if tokens <= capacity and cache <= MOST_CACHE and rows * heads * tokens * (prefix + capacity) <= \
                    MOST_SCORES // 8:
                return _prefix(None, dtype, rows, tokens, heads, kv, dim, prefix, capacity)
        else:
            layers, rows = _log(rng, 1, 32), _log(rng, 1, 8)
            budget = _log(rng, 32, 4096)
            longest = budget + (rng.randint(1, 4) if kind == "step" else _log(rng, 8, 4096))
            sinks = rng.choice([0, 1, 4])
            recent = min(budget - sinks, rng.choice([0, 16, budget // 4, budget // 2]))
            if 2 * layers * rows * kv * longest * dim * BYTES[dtype] <= MOST_CACHE:
                return _evict(None, dtype, layers, rows, kv, dim, longest, max(1, longest - rng.randint(0, 8)), budget,
                              sinks, recent)


def _spread(low, high, n, g):
    """n lengths from low to high, evenly spread, in an order made from the generator."""
    v = torch.linspace(low, high, n, dtype=torch.float64).round().to(torch.int32)
    return v[torch.randperm(n, generator=g)].cuda()


def _rows_of(case):
    """A window case's rows as (lowest start, highest start, shortest, longest): caches hold from half their
    capacity up to all of it; fused prompts are padded in front to the longest, by up to half."""
    c, n = case["capacity"], case["tokens"]
    if not case["ragged"]:
        return 0, 0, c, c
    return (0, c // 2, c, c) if case["fused"] else (0, 0, max(n, (c + 1) // 2), c)


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g, h = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "evict":
        L, R, H, C, D = (case[k] for k in ("layers", "rows", "kv_heads", "capacity", "head_dim"))
        s["keys"] = _normal((L, R, H, C, D), g, dtype)
        s["values"] = _normal((L, R, H, C, D), g, dtype)
        # Accumulated weights are heavy-tailed: a few slots hold most of the mass.
        s["weights"] = torch.exp(1.5 * torch.randn((L, R, H, C), generator=g, device="cuda"))
        # Token positions of the slots: what earlier evictions left, out of order.
        s["positions"] = torch.argsort(torch.rand((L, R, H, C), generator=g, device="cuda"), -1).to(torch.int32)
        s["lengths"] = _spread(case["shortest"], C, R, h)
        return s
    R, n, H, K, C, D = (case[k] for k in ("rows", "tokens", "heads", "kv_heads", "capacity", "head_dim"))
    lean = torch.randn((D,), generator=g, device="cuda")  # what queries have in common with the first tokens' keys
    if case["op"] == "window" and case["fused"]:
        x = torch.randn((R, n, (H + 2 * K) * D), generator=g, device="cuda")
        x[:, :, :H * D] += 0.5 * lean.repeat(H)
        x[:, 0, H * D:(H + K) * D] += lean.repeat(K)
        x = x.to(dtype)
        s["q"] = x[:, :, :H * D].unflatten(2, (H, D))
        s["keys"] = x[:, :, H * D:(H + K) * D].unflatten(2, (K, D)).transpose(1, 2)
        s["values"] = x[:, :, (H + K) * D:].unflatten(2, (K, D)).transpose(1, 2)
    else:
        s["q"] = (torch.randn((R, n, H, D), generator=g, device="cuda") + 0.5 * lean).to(dtype)
        k = torch.randn((R, K, C, D), generator=g, device="cuda")
        if case["op"] == "window":
            k[:, :, :max(1, case["sinks"])] += lean
        s["keys"] = k.to(dtype)
        s["values"] = _normal((R, K, C, D), g, dtype)
    if case["op"] == "window":
        first, last, shortest, longest = _rows_of(case)
        s["starts"] = _spread(first, last, R, h) if last else None
        s["lengths"] = _spread(shortest, longest, R, h) if shortest < longest else None
        if case["weigh"]:
            s["weights"] = torch.rand((R, K, C), generator=g, device="cuda")
    else:
        p = torch.randn((K, case["prefix"], D), generator=g, device="cuda")
        p[:, :1] += lean
        s["prefix_keys"] = p.to(dtype)
        s["prefix_values"] = _normal((K, case["prefix"], D), g, dtype)
        s["lengths"] = _spread(max(n, C // 2), C, R, h)
    return s


def _package():
    from __graft_entry__ import load_package
    return load_package()


def run(state):
    if own:
        return _own(state)
    return {"window": _plain_window, "prefix": _plain_prefix, "evict": _plain_evict}[state["op"]](state)


_sv = []


def _own(s):
    if not _sv:
        _sv.append(_package())
    sv = _sv[0]
    if s["op"] == "window":
        w = s.get("weights")
        out = sv.window_attention(s["q"], s["keys"], s["values"], s["lengths"], starts=s["starts"], window=s["window"],
                                  sinks=s["sinks"], weights=w)
        return {"out": out} if w is None else {"out": out, "weights": w}
    if s["op"] == "prefix":
        return {"out": sv.prefix_attention(s["q"], s["prefix_keys"], s["prefix_values"], s["keys"], s["values"],
                                           s["lengths"])}
    o = sv.kv_evict(s["keys"], s["values"], s["weights"], s["positions"], s["lengths"], s["budget"],
                    sinks=s["sinks"], recent=s["recent"])
    return {"keys": s["keys"], "values": s["values"], **o}


def _softmax(x, see):
    x = torch.where(see, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    t = e.sum(-1, keepdim=True)
    return e / torch.where(t > 0, t, 1.0)


def _at(lengths, rows, n, capacity, device):
    """Positions of the queries, [rows, 1, 1, n, 1]: they stand last in their rows."""
    i = torch.arange(n, device=device)
    at = i.expand(rows, n) + (capacity - n) if lengths is None else lengths[:, None] - n + i
    return at[:, None, None, :, None]


def _plain_window(s):
    q, k, v = s["q"].float(), s["keys"].float(), s["values"].float()
    R, n, H, D = q.shape
    K, C = k.shape[1], k.shape[2]
    x = q.reshape(R, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(R, K, H // K * n, D)
    scores = (torch.matmul(x, k.transpose(2, 3)) * D ** -0.5).view(R, K, H // K, n, C)
    slot = torch.arange(C, device=q.device)
    at = _at(s["lengths"], R, n, C, q.device)
    first = 0 if s["starts"] is None else s["starts"].view(R, 1, 1, 1, 1)
    see = (slot <= at) & (slot >= first)
    if s["window"]:
        see = see & ((slot > at - s["window"]) | (slot < first + s["sinks"]))
    p = _softmax(scores, see)
    o = torch.matmul(p.view(R, K, H // K * n, C), v).view(R, K, H // K, n, D).permute(0, 3, 1, 2, 4)
    out = o.reshape(R, n, H, D).to(s["q"].dtype)
    if "weights" not in s:
        return {"out": out}
    s["weights"] += p.sum((2, 3))
    return {"out": out, "weights": s["weights"]}


def _plain_prefix(s):
    q, k, v = s["q"].float(), s["keys"].float(), s["values"].float()
    pk, pv = s["prefix_keys"].float(), s["prefix_values"].float()
    R, n, H, D = q.shape
    K, C, P = k.shape[1], k.shape[2], pk.shape[1]
    x = q.view(R, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(R, K, H // K * n, D)
    a = torch.matmul(x, pk.transpose(1, 2)).view(R, K, H // K, n, P)
    b = torch.matmul(x, k.transpose(2, 3)).view(R, K, H // K, n, C)
    at = _at(s["lengths"], R, n, C, q.device)
    see = (torch.arange(P + C, device=q.device) - P) <= at
    p = _softmax(torch.cat([a, b], -1) * D ** -0.5, see | (torch.arange(P + C, device=q.device) < P)) \
        .view(R, K, H // K * n, P + C)
    o = torch.matmul(p[..., :P], pv) + torch.matmul(p[..., P:], v)
    return {"out": o.view(R, K, H // K, n, D).permute(0, 3, 1, 2, 4).reshape(R, n, H, D).to(s["q"].dtype)}


def _plain_evict(s):
    w, pos, B = s["weights"], s["positions"], s["budget"]
    L, R, H, C = w.shape
    slot = torch.arange(C, device=w.device)
    valid = slot < s["lengths"][:, None, None]
    newest = torch.where(valid, pos, -1).amax(-1, keepdim=True)
    stays = (pos < s["sinks"]) | (pos > newest - s["recent"])
    rank = torch.where(stays, math.inf, torch.where(torch.isnan(w), -math.inf, w))
    # Heaviest first, ties to the lowest slot: a stable order of the valid slots, the others last.
    heavy = torch.argsort(rank, dim=-1, descending=True, stable=True)
    heavy = torch.gather(heavy, -1, torch.argsort((~valid.expand(w.shape)).gather(-1, heavy).int(), dim=-1, stable=True))
    place = torch.empty_like(heavy).scatter_(-1, heavy, slot.expand(w.shape).contiguous())
    kept = valid & (place < B)
    # Survivors past the budget take the evicted slots below it, both in slot order.
    comes = kept & (slot >= B)
    hole = ~kept & (slot < B) & valid
    free = torch.argsort(~hole, dim=-1, stable=True, descending=False)
    goes = torch.gather(free, -1, (comes.cumsum(-1) - 1).clamp_min(0))
    unit = torch.arange(L * R * H, device=w.device).view(L, R, H, 1)
    src, dst = (unit * C + slot)[comes], (unit * C + goes)[comes]
    ends = torch.minimum(s["lengths"], torch.tensor(B, device=w.device, dtype=torch.int32))
    out = {"lengths": ends}
    for name, t, rest in (("weights", w, 0.0), ("positions", pos, -1)):
        x = t.clone()
        x.view(-1)[dst] = x.view(-1)[src]
        out[name] = torch.where(slot < ends[:, None, None], x, torch.full_like(x, rest))
    for name in ("keys", "values"):
        x = s[name].view(L * R * H * C, -1)
        x[dst] = x[src]
        out[name] = s[name]
    return out


def work(case):
    e, D = BYTES[case["dtype"]], case["head_dim"]
    if case["op"] == "evict":
        L, R, H, C, B = (case[k] for k in ("layers", "rows", "kv_heads", "capacity", "budget"))
        lengths = torch.linspace(case["shortest"], C, R, dtype=torch.float64).round().tolist()
        cuts = [(n, max(0.0, n - B) / n) for n in lengths]
        moved = sum((n - B) * B / n for n, cut in cuts if cut)  # as many as lie past the budget by chance
        return {"bytes": L * H * (sum(8 * n + 8 * C for n in lengths) + moved * 4 * D * e), "flops": L * H * sum(lengths)}
    R, n, H, K, C = (case[k] for k in ("rows", "tokens", "heads", "kv_heads", "capacity"))
    ends = R * n * H * D * e * 2
    if case["op"] == "prefix":
        lengths = torch.linspace(max(n, C // 2), C, R, dtype=torch.float64).round()
        pairs = n * (R * case["prefix"] + float(lengths.sum())) - R * n * (n - 1) / 2
        return {"bytes": ends + 2 * K * D * e * (case["prefix"] + float(lengths.sum())), "flops": 4 * D * H * pairs}
    low, high, shortest, longest = _rows_of(case)
    start = torch.linspace(low, high, R, dtype=torch.float64).round()[:, None]
    at = torch.linspace(shortest, longest, R, dtype=torch.float64).round()[:, None] - n + torch.arange(n) - start
    w, k = case["window"] or C, torch.tensor(float(case["sinks"]))
    seen, low = (at + 1).clamp(min=0), (at - w + 1).clamp(min=0)
    pairs = float((seen - low + torch.minimum(low, k)).sum())
    slots = float((seen[:, -1] - low[:, 0] + torch.minimum(low[:, 0], k)).sum())
    return {"bytes": ends + 2 * K * D * e * slots + (8 * K * slots if case["weigh"] else 0), "flops": 4 * D * H * pairs}


def exact(case, seed):
    """The operators' definitions in 64 bits, one row and key/value head at a time."""
    s = prepare(case, seed)
    if case["op"] == "evict":
        return None  # moves values, computes none
    q = s["q"].double()
    R, n, H, D = q.shape
    K, G, C = case["kv_heads"], H // case["kv_heads"], case["capacity"]
    out = torch.zeros_like(q)
    acc = s["weights"].double() if "weights" in s else None
    for r in range(R):
        end = C if s["lengths"] is None else int(s["lengths"][r])
        start = 0 if s.get("starts") is None else int(s["starts"][r])
        for h in range(K):
            keys, vals = s["keys"][r, h, :end].double(), s["values"][r, h, :end].double()
            before = 0
            if case["op"] == "prefix":
                before = case["prefix"]
                keys = torch.cat([s["prefix_keys"][h].double(), keys])
                vals = torch.cat([s["prefix_values"][h].double(), vals])
            if not len(keys):
                continue
            j = torch.arange(len(keys), device=q.device) - before
            i = torch.arange(n, device=q.device)[:, None] + (end - n)
            hidden = j > i
            if case["op"] == "window" and case["window"]:
                hidden |= (j <= i - case["window"]) & (j >= start + case["sinks"])
            hidden = (hidden & (j >= 0)) | ((j >= 0) & (j < start))
            for g in range(h * G, (h + 1) * G):
                z = (q[r, :, g] @ keys.T).mul_(1 / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
                out[r, :, g] = p @ vals
                if acc is not None:
                    acc[r, h, :end] += p.sum(0)
    return {"out": out} if acc is None else {"out": out, "weights": acc}
