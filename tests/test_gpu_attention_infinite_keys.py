"""Accumulated weights where a key holds an infinity that gives every query that sees it a
score of minus infinity: a weight of zero, as in the formula, and no effect on other slots."""
import pytest
import torch

from _attention_ref import U, attention, check
from test_gpu_attention import i32, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 1, 4, 2, 64, 30, 0, 0), (3, 5, 8, 2, 128, 40, 0, 0), (2, 61, 3, 1, 72, 90, 0, 0),
                                   (2, 84, 5, 5, 8, 138, 14, 64), (1, 300, 7, 1, 64, 310, 0, 0)])
def test_scores_of_minus_infinity(sv, shape, dtype):
    R, n, H, K, D, C, window, sinks = shape
    q, k, v = rand((R, n, H, D), 1, dtype), rand((R, K, C, D), 2, dtype), rand((R, K, C, D), 3, dtype)
    q[..., 5] = q[..., 5].abs() + 0.25  # finite with every other key; with -inf in this dimension, never +inf or NaN
    lengths = i32([C - r for r in range(R)])
    hidden = [0, C // 2, C - n, C - R]
    before, clean = k.clone(), k.clone()
    clean[:, :, hidden, 5] = -60000.0  # a weight of zero in any precision
    k[:, :, hidden, 5] = -torch.inf
    want, _, wts, _ = attention(q, clean, v, lengths, None, window, sinks)
    # Bounds of _attention_ref, of the scores that are left: no larger than those of the keys before.
    big = max(float((q[r].transpose(0, 1).abs().double() @ before[r, h].abs().double().T).max()) for r in range(R)
              for h in range(K)) * D ** -0.5
    err = 2 * (D + 8) * 2.0 ** -24 * big + 2.0 ** -20
    u = U[dtype]
    tol = (u + (0.0 if dtype == torch.float32 else u) + err + (C * 2.0 ** -25 if dtype == torch.float16 else 0.0)) * \
        v.abs().max().double()
    w = torch.zeros((R, K, C), device=DEV)
    got = sv.window_attention(q, k, v, lengths, window=window, sinks=sinks, weights=w)
    check(got, want, tol, "out")
    check(w, wts, (err + 2.0 ** -22 + 2.0 ** -23) * wts + 1e-30, "weights")
    assert (w[:, :, hidden] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 45])
def test_a_row_of_nothing_else(sv, dtype, n):
    """Rows whose every slot has that score: zeros, as rows that see nothing."""
    q, k, v = rand((1, n, 6, 64), 4, dtype).abs() + 0.25, rand((1, 2, 50, 64), 5, dtype), rand((1, 2, 50, 64), 6, dtype)
    k[:, 0, :, 7] = -torch.inf
    w = torch.zeros((1, 2, 50), device=DEV)
    got = sv.window_attention(q, k, v, weights=w)
    assert (got[:, :, :3] == 0).all() and (w[:, 0] == 0).all()
    want, tol, wts, wtol = attention(q[:, :, 3:], k[:, 1:], v[:, 1:])
    check(got[:, :, 3:], want, tol, "the other head")
    check(w[:, 1:], wts, wtol + 2.0 ** -23 * wts + 1e-30, "its weights")
