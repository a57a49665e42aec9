"""kv_quantize where lanes of a warp go different ways, and where a float16 pair hangs on bits that are far apart, against
the format in exact fractions."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from _records_ref import MOST, dims, encode, group, place, record, same_values

DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.gpu
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


def half(x):
    """The float16 next to a fraction, ties to the even one."""
    y = np.float16(float(x))
    near = [np.nextafter(y, np.float16(-np.inf)), y, np.nextafter(y, np.float16(np.inf))]
    return min((z for z in near if np.isfinite(z)), key=lambda z: (abs(Fraction(float(z)) - x), int(z.view(np.uint16)) & 1))


def encode_exactly(x):
    """Records of finite float32 rows [rows, D] in fractions."""
    D = x.shape[-1]
    P, G, (w, n) = dims(D), group(D), place(D)
    words, pairs = np.zeros((len(x), P // 8), np.uint32), np.zeros((len(x), 8), np.float16)
    for r, row in enumerate(x):
        for k, d0 in enumerate(range(0, D, G)):
            v = [Fraction(max(-MOST, min(MOST, float(y)))) for y in row[d0:d0 + G]]
            s = half((max(v) - min(v)) / 15)
            s_ = Fraction(float(s))
            m = half(min(v) + 8 * s_)
            pairs[r, 2 * k], pairs[r, 2 * k + 1] = s, m
            for d, y in enumerate(v, d0):
                c = 8 + (round((y - Fraction(float(m))) / s_) if s_ else 0)  # (round: ties to the even one)
                words[r, w[d]] |= np.uint32(max(0, min(15, c)) << int(4 * n[d]))
    return np.concatenate([words.view(np.uint8), pairs.view(np.uint8)], -1)


def test_halves_of_fractions():
    g = np.random.default_rng(1)
    for x in np.concatenate([g.standard_normal(300) * 2.0 ** g.integers(-26, 13, 300), [2.0 ** -25, 3 * 2.0 ** -25, 0.0, 60000.0]]):
        assert half(Fraction(float(x))) == np.float16(x)
    tie = Fraction(1) + Fraction(1, 2048)
    assert half(tie) == 1 and half(tie + Fraction(1, 10 ** 40)) == np.float16(1 + 2.0 ** -10)
    x = g.standard_normal((6, 72)).astype(np.float32)
    assert np.array_equal(encode_exactly(x), encode(x.astype(np.float64)))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_scales_whose_border_hangs_on_a_tiny_extreme(sv, D):
    """Extremes that differ by fifteen times a border of float16, but for something below 2^-60 of it."""
    g = np.random.default_rng(2)
    rows = []
    for _ in range(300):
        h = np.float32(15 * (1024 + g.integers(0, 1024) + 0.5) * 2.0 ** g.integers(-20, 0))
        x = (h * g.random(D)).astype(np.float32)
        x[::8] = np.float32(g.choice([1e-30, -1e-30, 1e-44, -1e-44, -1e-12, 0.0]))
        x[3::16] = h
        rows.append(x if g.random() < 0.5 else -x)
    # A border among float16's subnormals too.
    x = np.full(D, 15 * 2.0 ** -25, np.float32)
    x[::8] = 1e-40
    rows += [x, -x]
    x = np.stack(rows)
    assert (encode(x.astype(np.float64)) != encode_exactly(x)).any()  # 64 bits do not do
    c = torch.zeros((len(x), 1, 1, record(D)), dtype=torch.uint8, device=DEV)
    sv.kv_quantize(torch.from_numpy(x).to(DEV)[:, None, None], None, c, None)
    assert same_values(c[:, 0, 0], encode_exactly(x), D)
