"""kv_quantize where lanes of a warp go different ways."""
import pytest
import torch

from _records_ref import encode, record, same_values

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 40, 64, 72, 96, 120, 128])
def test_groups_of_all_kinds_in_one_warp(sv, D, dtype):
    """Ordinary groups, ones far from zero, past the range, constant and not finite, side by side in every order, with
    tokens that are left out and lanes without dimensions."""
    g = torch.Generator().manual_seed(D)
    R, K, n, C = 3, 2, 37, 30
    x = torch.randn((R, K, n, D), generator=g)
    kind = torch.randint(0, 6, (R, K, n, (D + 15) // 16), generator=g).repeat_interleave(16, -1)[..., :D]
    x = torch.where(kind == 1, 500 + x * 2.0 ** -6, x)
    x = torch.where(kind == 2, x * 40000.0, x)
    x = torch.where(kind == 3, 1.5, x)
    x = torch.where((kind == 4) & (x > 1), float("nan"), x)
    x = torch.where((kind == 5) & (x > 1), float("inf"), x)
    x = x.to(dtype)
    c = torch.full((R, K, C, record(D)), 7, dtype=torch.uint8, device=DEV)
    lengths = torch.tensor([30, 11, 0], dtype=torch.int32, device=DEV)
    sv.kv_quantize(x.to(DEV), None, c, None, lengths)
    want = torch.full((R, K, C, record(D)), 7, dtype=torch.uint8).numpy()
    for r, end in enumerate([30, 11, 0]):
        if end:
            want[r, :, :end] = encode(x[r, :, n - end:].double().numpy())
    assert same_values(c, want, D)
