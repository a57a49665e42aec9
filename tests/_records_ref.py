"""The cache held in 4 bits in 64-bit arithmetic: records written and read by the format's
words, attention over them, and how far a kernel may be from it.

Error bound of the attention, as in _attention_ref, with two more roundings: the 16-bit
kernels may hold each key and value once in the inputs' type (unit roundoff u = 2^-8 for
bfloat16, 2^-11 for float16; float16 below 2^-14 absolutely, 2^-25).  With S = sum_d |q_d
k_d| |scale| a score is off by at most (u + (D + 8) 2^-24) S, a weight relatively by at
most exp(twice that) - 1 + 2^-20, and with A = sum_j p_j |v_j| the output by
  u |o| + (2 u + e) A + 2^-24 sum_j |v_j| + 2^-25 (16-bit types; u = 0 in the middle terms for float32).
"""
import numpy as np
import torch

from _attention_ref import U, visible

MOST = 32768.0


def dims(D):
    return (D + 31) // 32 * 32


def group(D):
    return 32 if D > 64 else 16


def record(D):
    return dims(D) // 2 + 16


def place(D):
    """(word, nibble) of each dimension, padded ones included."""
    d = np.arange(dims(D))
    i, e, t, a, b = d >> 5, d >> 4 & 1, d >> 2 & 3, d >> 1 & 1, d & 1
    return t * (dims(D) // 32) + i, 4 * b + 2 * e + a


def encode(x):
    """Records uint8 [..., record] of float64 values [..., D]."""
    D = x.shape[-1]
    P, G = dims(D), group(D)
    code = np.zeros(x.shape[:-1] + (P,), np.uint32)
    pairs = np.zeros(x.shape[:-1] + (8,), np.float16)
    with np.errstate(invalid="ignore"):
        for k, d in enumerate(range(0, D, G)):
            y = np.asarray(x[..., d:d + G], np.float64)
            bad = ~np.isfinite(y).all(-1)
            y = np.clip(np.where(np.isfinite(y), y, 0.0), -MOST, MOST)
            lo = y.min(-1)
            s = ((y.max(-1) - lo) / 15).astype(np.float16)
            m = (lo + 8 * s.astype(np.float64)).astype(np.float16)
            s64, m64 = s.astype(np.float64)[..., None], m.astype(np.float64)[..., None]
            c = np.rint(np.divide(y - m64, s64, out=np.zeros_like(y), where=s64 != 0)) + 8
            code[..., d:min(d + G, D)] = np.where(bad[..., None], 0, np.clip(c, 0, 15)).astype(np.uint32)
            pairs[..., 2 * k] = np.where(bad, np.float16(np.nan), s)
            pairs[..., 2 * k + 1] = np.where(bad, np.float16(np.nan), m)
    words = np.zeros(x.shape[:-1] + (P // 8,), np.uint32)
    w, n = place(D)
    for d in range(D):
        words[..., w[d]] |= code[..., d] << np.uint32(4 * n[d])
    return np.concatenate([words.view(np.uint8), pairs.view(np.uint8)], -1)


def decode(records, D):
    """What records (uint8 tensor [..., record]) stand for, float64 [..., D] on their device."""
    r = records.cpu().numpy()
    P, G = dims(D), group(D)
    words = np.ascontiguousarray(r[..., :P // 2]).view(np.uint32)
    pairs = np.ascontiguousarray(r[..., P // 2:]).view(np.float16).astype(np.float64)
    w, n = place(D)
    x = np.empty(r.shape[:-1] + (D,))
    for d in range(D):
        c = (words[..., w[d]] >> np.uint32(4 * n[d]) & np.uint32(15)).astype(np.float64)
        x[..., d] = pairs[..., 2 * (d // G) + 1] + pairs[..., 2 * (d // G)] * (c - 8)
    return torch.from_numpy(x).to(records.device)


def same_values(got, want, D):
    """Whether two arrays of records hold the same codes, and pairs of the same value (0 and -0 alike)."""
    g, w = got.cpu().numpy(), np.asarray(want)
    c = dims(D) // 2
    pg = np.ascontiguousarray(g[..., c:]).view(np.float16)
    pw = np.ascontiguousarray(w[..., c:]).view(np.float16)
    return (g[..., :c] == w[..., :c]).all() and ((pg == pw) | (np.isnan(pg) & np.isnan(pw))).all()


def attention(q, keys, values, lengths=None, starts=None, window=0, sinks=0, scale=None):
    """(out, tolerance, weights, weight tolerance) in float64; keys / values float64 [R, K, C, D] as decoded."""
    R, n, H, D = q.shape
    K, C = keys.shape[1], keys.shape[2]
    G = H // K
    scale = D ** -0.5 if scale is None else scale
    dev = q.device
    out = torch.zeros((R, n, H, D), dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    wts = torch.zeros((R, K, C), dtype=torch.float64, device=dev)
    wtol = torch.zeros_like(wts)
    u = U[q.dtype]
    short = q.dtype != torch.float32
    u16 = u if short else 0.0
    for r in range(R):
        end = C if lengths is None else min(max(int(lengths[r]), 0), C)
        start = 0 if starts is None else min(max(int(starts[r]), 0), end)
        see = visible(n, C, end, start, window, sinks, dev)
        any_row = see.any(0)[:, None]
        k = torch.where(any_row[None], keys[r], 0.0)
        v = torch.where(any_row[None], values[r], 0.0)
        x = q[r].double().view(n, K, G, D).permute(1, 2, 0, 3)  # [K, G, n, D]
        s = (x @ k[:, None].transpose(2, 3)) * scale
        s = torch.where(see, s, -torch.inf)
        m = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(m == -torch.inf, 0.0, m))
        t = e.sum(-1, keepdim=True)
        p = e / torch.where(t > 0, t, 1.0)
        big = torch.where(see, (x.abs() @ k.abs()[:, None].transpose(2, 3)) * abs(scale), 0.0).amax(-1, keepdim=True)
        err = torch.expm1(2 * (u16 + (D + 8) * 2.0 ** -24) * big) + 2.0 ** -20
        o = p @ v[:, None]
        b = u * o.abs() + (2 * u16 + err) * (p @ v.abs()[:, None]) + 1e-30
        if short:
            b += 2.0 ** -24 * (see.double() @ v.abs())[:, None] + 2.0 ** -25
        out[r] = o.permute(2, 0, 1, 3).reshape(n, H, D)
        tol[r] = b.permute(2, 0, 1, 3).reshape(n, H, D)
        wts[r] = p.sum((1, 2))
        wtol[r] = (p * (err + 2.0 ** -22)).sum((1, 2)) + 1e-30
    return out, tol, wts, wtol
