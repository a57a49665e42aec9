"""Attention over a cache in 64 bits, and how far a kernel may be from it.

Error bound, derived from the arithmetic the kernels state (all scores, maxima and
sums in f32, products of the inputs exact or f32):
  * a score is off by at most (D + 8) 2^-24 sum_d |q_d k_d| |scale|, so a softmax
    weight by twice the largest such error, relatively (numerator and denominator);
    exp2 and the sums over the slots add a few 2^-24 each, 2^-20 covers them;
  * the 16-bit kernels round each weight once to the inputs' type (relative error at
    most the unit roundoff u = 2^-p for p significant bits: 2^-8 for bfloat16, 2^-11
    for float16; float16 weights below 2^-14 of the largest absolutely, 2^-25) and every
    kernel rounds the output once (u |o|).
With A = sum_j p_j |v_j| the output's error is at most
  u |o| + (u_weight + e) A + a sum_j |v_j|,  e = 2 (D + 8) 2^-24 S + 2^-20.
"""
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def visible(n, lo_slot, end, start, window, sinks, device):
    """[n, slots] of a row's own slots, and the queries' positions."""
    p = torch.arange(n, device=device)[:, None] + (end - n)
    j = torch.arange(lo_slot, device=device)[None, :]
    see = (j <= p) & (j >= start)
    if window:
        see &= (j > p - window) | (j < start + sinks)
    return see


def attention(q, keys, values, lengths=None, starts=None, window=0, sinks=0, scale=None, prefix=None):
    """(out, tolerance, weights, weight tolerance) in float64.  q [R, n, H, D], keys /
    values [R, K, C, D], prefix (keys, values) [K, P, D] or None."""
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
    uw = 0.0 if q.dtype == torch.float32 else u
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    for r in range(R):
        end = C if lengths is None else min(max(int(lengths[r]), 0), C)
        start = 0 if starts is None else min(max(int(starts[r]), 0), end)
        see = visible(n, C, end, start, window, sinks, dev)
        P = 0 if prefix is None else prefix[0].shape[1]
        if P:
            see = torch.cat([torch.ones((n, P), dtype=torch.bool, device=dev), see], 1)
        any_row = see.any(0)  # slots nobody sees may hold anything
        for h in range(K):
            k, v = keys[r, h].double(), values[r, h].double()
            if P:
                k, v = torch.cat([prefix[0][h].double(), k]), torch.cat([prefix[1][h].double(), v])
            k = torch.where(any_row[:, None], k, 0.0)
            v = torch.where(any_row[:, None], v, 0.0)
            for g in range(h * G, (h + 1) * G):
                x = q[r, :, g].double()
                s = (x @ k.T) * scale
                m = torch.where(see, s, -torch.inf).amax(1, keepdim=True)
                m = torch.where(m == -torch.inf, 0.0, m)
                e = torch.where(see, torch.exp(s - m), 0.0)
                t = e.sum(1, keepdim=True)
                p = e / torch.where(t > 0, t, 1.0)
                big = torch.where(see, (x.abs() @ k.abs().T) * abs(scale), 0.0).amax(1, keepdim=True)
                err = 2 * (D + 8) * 2.0 ** -24 * big + 2.0 ** -20
                o = p @ v
                out[r, :, g] = o
                tol[r, :, g] = u * o.abs() + (uw + err) * (p @ v.abs()) + tiny * (see.double() @ v.abs()) + 1e-30
                w = p[:, P:]
                wts[r, h] += w.sum(0)
                wtol[r, h] += (w * (err + 2.0 ** -22)).sum(0)
    return out, tol, wts, wtol


def check(got, want, tol, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs()
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"
