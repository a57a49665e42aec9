"""The tile kernel's bounded waits: the test hook makes those of one key/value head's blocks
run out.  Their outputs are NaN and their rows report it, whichever head it was; the others
are right, and so are the next call's."""
import pytest
import torch

from _attention_ref import attention, check
from test_gpu_attention import i32, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"

# rows, tokens, heads, kv_heads, head_dim, capacity: one tile, split; two tiles; halves.  A block has one piece.
SHAPES = [(3, 40, 8, 4, 64, 600), (9, 500, 8, 4, 128, 500), (20, 20, 8, 4, 64, 1700)]


@pytest.mark.parametrize("head", [0, 2, 3])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_wait_that_runs_out(sv, shape, head):
    R, n, H, K, D, C = shape
    q, k, v = rand((R, n, H, D), 1, torch.float16), rand((R, K, C, D), 2, torch.float16), rand((R, K, C, D), 3, torch.float16)
    lengths = i32([C] * (R - 1) + [C + 1])  # the last row's is clamped
    want, tol, _, _ = attention(q, k, v)
    status = i32([-1] * R)
    sv._lib.lib().sv_test_attention_timeout(head)
    got = sv.window_attention(q, k, v, lengths, status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [sv._lib.ST_TIMEOUT] * R
    mine = torch.arange(H, device=DEV) // (H // K) == head
    assert torch.isnan(got[:, :, mine]).all()
    check(got[:, :, ~mine], want[:, :, ~mine], tol[:, :, ~mine], "the other heads")
    got = sv.window_attention(q, k, v, lengths, status=status)
    assert status.tolist() == [0] * (R - 1) + [sv._lib.ST_LENGTH]
    check(got, want, tol, "the next call")


def test_nothing_else_is_waited_for(sv):
    """A block of one tile: its other product warp has no products to drain and is not waited for."""
    R, n, H, K, D, C = SHAPES[0]
    q, k = rand((R, n, H, D), 1, torch.float16), rand((R, K, C, D), 2, torch.float16)
    sv.window_attention(q, k, k)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    sv._lib.lib().sv_test_attention_timeout(1)
    start.record()
    got = sv.window_attention(q, k, k)
    end.record()
    end.synchronize()
    assert torch.isnan(got[:, :, 2:4]).all()
    assert start.elapsed_time(end) < 500  # ms: waits of 2 ms each, none of the 1 s of a barrier that nobody reaches
