"""quantized_attention within bounds that count its roundings and no others: keys are not rounded to the inputs' type.

Scores are formed from codes c (0..15), scale s and middle m as sum q s c + sum q (m - 8 s), in sums of 17 terms that a tensor
core may truncate below 2^-24 of the largest: off by at most 2^-19 S', S' = |scale| sum_d |q_d| (23 s_d + |m_d|) (float32
queries: 22 bits of them, within that).  Calls past 64 query rows per key/value head take the keys from float16, one for
bfloat16 queries (2^-11 S, S = |scale| sum |q k|), two for float16, float16's subnormals apart (2^-25 |scale| sum |q|).  A
weight is relatively off by err = exp(twice the largest of these) - 1 + 2^-20 + C / 4 2^-24 (f32 sums of the slots that
one thread adds).  With A = sum p |v| the output is off by
  u |o| + err A                                                           float32
  u |o| + (2^-11 + w + err) A + 2^-32 sum |v| + 2^-24                     16-bit: values in float16,
weights in float16 (w = 2^-11; float16 calls: in two, 2^-21), held to 2^-32 of the heaviest."""
import numpy as np
import pytest
import torch

from _attention_ref import U, check, visible
from _records_ref import decode, dims, group
from test_gpu_quantized_attention import DEV, DTYPES, PROMPT, TOKEN, cache, i32, lengths_for, rand
from test_gpu_quantized_exactness import alternating

pytestmark = pytest.mark.gpu


def spread(records, D):
    """23 s + |m| of each dimension, float64 [..., D]."""
    pairs = np.ascontiguousarray(records.cpu().numpy()[..., dims(D) // 2:]).view(np.float16).astype(np.float64)
    d = np.arange(D) // group(D)
    return torch.from_numpy(23 * pairs[..., 2 * d] + np.abs(pairs[..., 2 * d + 1])).to(records.device)


def bounded(q, ck, cv, lengths, window, sinks, scale=None):
    """(out, bound, weights, their bound) in float64."""
    R, n, H, D = q.shape
    K, C = ck.shape[1], ck.shape[2]
    G = H // K
    scale = D ** -0.5 if scale is None else scale
    short, many = q.dtype != torch.float32, n * G > (32 if q.dtype == torch.float32 else 64)
    keys, values, wide = decode(ck, D), decode(cv, D), spread(ck, D)
    out = torch.zeros((R, n, H, D), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    wts = torch.zeros((R, K, C), dtype=torch.float64, device=DEV)
    wtol = torch.zeros_like(wts)
    for r in range(R):
        end = C if lengths is None else int(lengths[r])
        see = visible(n, C, end, 0, window, sinks, DEV)
        x = q[r].double().view(n, K, G, D).permute(1, 2, 0, 3)
        k, v = keys[r][:, None], values[r][:, None]
        s = torch.where(see, (x @ k.transpose(2, 3)) * scale, -torch.inf)
        p = torch.softmax(s, -1)
        e = 2.0 ** -19 * (x.abs() @ wide[r][:, None].transpose(2, 3))
        if short and many:
            e += 2.0 ** -25 * x.abs().sum(-1, keepdim=True)
            if q.dtype == torch.bfloat16:
                e += 2.0 ** -11 * (x.abs() @ k.abs().transpose(2, 3))
        e = torch.where(see, e * abs(scale), 0.0).amax(-1, keepdim=True)
        err = torch.expm1(2 * e) + 2.0 ** -20 + C / 4 * 2.0 ** -24
        o, A = p @ v, p @ v.abs()
        b = U[q.dtype] * o.abs() + err * A + 1e-30  # (not zero over zero)
        if short:
            b += (2.0 ** -11 + (2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -21)) * A
            b += 2.0 ** -32 * (see.double() @ v.abs()) + 2.0 ** -24
        out[r] = o.permute(2, 0, 1, 3).reshape(n, H, D)
        tol[r] = b.permute(2, 0, 1, 3).reshape(n, H, D)
        wts[r] = p.sum((1, 2))
        wtol[r] = (p * err).sum((1, 2)) + 1e-30
    return out, tol, wts, wtol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TOKEN + PROMPT)
def test_within_the_roundings(sv, shape, dtype):
    R, n, H, K, D, C, window, sinks = shape
    q = rand((R, n, H, D), 1, dtype, 1.5)
    ck, cv = cache(sv, (R, K, C, D), 2, shift=0.3), cache(sv, (R, K, C, D), 3)
    for lengths in (None, i32(lengths_for(R, n, C))):
        w = torch.zeros((R, K, C), device=DEV)
        want, tol, wts, wtol = bounded(q, ck, cv, lengths, window, sinks)
        check(sv.quantized_attention(q, ck, cv, lengths, window=window, sinks=sinks), want, tol, f"{shape} {lengths}")
        got = sv.quantized_attention(q, ck, cv, lengths, window=window, sinks=sinks, weights=w)
        check(got, want, tol, f"{shape} {lengths} with weights")
        check(w, wts, wtol, f"{shape} {lengths} weights")
        if dtype != torch.bfloat16 or n * (H // K) <= 64:  # the bound tells an output from none
            assert (want.abs() <= tol).double().mean() < 0.1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 4, 40])
def test_large_queries_and_keys_far_from_zero(sv, dtype, n):
    R, H, K, D, C = 2, 8, 2, 128, 300
    q = rand((R, n, H, D), 4, dtype, 4.0)
    ck, cv = cache(sv, (R, K, C, D), 5, shift=4.0), cache(sv, (R, K, C, D), 6)
    want, tol, _, _ = bounded(q, ck, cv, None, 0, 0)
    check(sv.quantized_attention(q, ck, cv), want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,n,H,K,D,C", [(2, 1, 4, 1, 128, 600), (2, 1, 36, 4, 64, 600), (3, 5, 36, 4, 128, 400),
                                         (2, 90, 8, 2, 64, 700)])
def test_keys_that_the_inputs_type_does_not_hold(sv, dtype, R, n, H, K, D, C):
    """Keys rounded to the inputs' type would weigh all slots alike."""
    q, scale, ck, cv, share, _, bound = alternating(sv, dtype, R, n, H, K, D, C, fine=dtype != torch.bfloat16 or n * H // K <= 64)
    want = share[None, :, None, None].expand(q.shape)
    tol = want * (bound + U[dtype] + (2 * 2.0 ** -11 if dtype != torch.float32 else 0.0))
    check(sv.quantized_attention(q, ck, cv, scale=scale), want, tol)
    if dtype != torch.float32:
        k = decode(ck[:1, :1], D).to(dtype).double()[0, 0]
        rounded = torch.softmax(q[0, -1, 0].double() @ k.T * scale, -1)[::2].sum()
        assert (rounded - want[0, -1, 0, 0]).abs() > 10 * tol[0, -1, 0, 0]
