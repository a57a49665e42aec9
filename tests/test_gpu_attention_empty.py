"""Calls without queries or without slots: the result's shape, `out` itself, every status."""
import pytest
import torch

from _attention_ref import attention, check
from test_gpu_attention import i32, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 1, 4, 64), (3, 20, 4, 64), (3, 4, 64)])
def test_no_slots(sv, shape, dtype):
    q, k = rand(shape, 1, dtype), rand((3, 2, 0, 64), 2, dtype)
    pk, pv = rand((2, 77, 64), 3, dtype), rand((2, 77, 64), 4, dtype)
    one = rand((3, 2, 1, 64), 5, dtype)
    whole = q if q.dim() == 4 else q[:, None]
    want, tol, _, _ = attention(whole, one, one, [0, 0, 0], prefix=(pk, pv))
    for lengths, states in ((None, [0, 0, 0]), (i32([0, 1, -1]), [0, 8, 8])):
        for out in (None, torch.full(shape, 7, dtype=dtype, device=DEV)):
            status = i32([-1, -1, -1])
            got = sv.window_attention(q, k, k, lengths, out=out, status=status)
            assert got.shape == q.shape and (got == 0).all() and status.tolist() == states
            assert out is None or got is out
            status = i32([-1, -1, -1])
            got = sv.prefix_attention(q, pk, pv, k, k, lengths, out=out, status=status)
            assert got.shape == q.shape and status.tolist() == states
            assert out is None or got is out
            check(got.view(whole.shape), want, tol, "prefix alone")
    status = i32([-1, -1, -1])
    sv.window_attention(q, k, k, starts=i32([0, 1, -2]), status=status)
    assert status.tolist() == [0, 8, 8]


def test_no_queries(sv):
    q, k = rand((3, 0, 4, 64), 6, torch.float16), rand((3, 2, 9, 64), 7, torch.float16)
    for lengths, starts, states in ((None, None, [0, 0, 0]), (i32([9, 10, -1]), None, [0, 8, 8]),
                                    (i32([5, 5, 5]), i32([5, 6, -1]), [0, 8, 8]), (None, i32([9, 10, 0]), [0, 8, 0])):
        status = i32([-1, -1, -1])
        assert sv.window_attention(q, k, k, lengths, starts=starts, status=status).shape == q.shape
        assert status.tolist() == states
        if starts is None:
            status = i32([-1, -1, -1])
            assert sv.prefix_attention(q, k[0], k[0], k, k, lengths, status=status).shape == q.shape
            assert status.tolist() == states
    with pytest.raises(RuntimeError):
        sv.window_attention(q, k, k, status=torch.zeros(2, dtype=torch.int32, device=DEV))
