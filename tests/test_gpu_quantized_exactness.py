"""quantized_attention where a small error of its own would show: structured inputs whose results follow from a few
exact numbers.  Keys that are constant within a group are held exactly (scale 0), so scores are known.  Bounds count
roundings: U of the output's type, half a step each; what a 16-bit call's tensor cores take is float16 (2^-11)."""
import math

import pytest
import torch

from _attention_ref import U, check
from _records_ref import attention, decode, record

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SHORT = [torch.float16, torch.bfloat16]


def rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def records(sv, x):
    c = torch.zeros(x.shape[:-1] + (record(x.shape[-1]),), dtype=torch.uint8, device=DEV)
    sv.kv_quantize(x, None, c, None)
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2, 3, 6, 16, 90])
@pytest.mark.parametrize("below", [5, 18, 40, 200])
def test_nan_under_a_small_weight(sv, dtype, n, below):
    """Values that stand for NaN make NaN of every query that sees their slot, however little it weighs there."""
    R, H, K, D, C = 1, 4, 2, 64, 320
    where = C - 2  # seen by the last two queries
    q = torch.ones((R, n, H, D), dtype=dtype, device=DEV)
    x, y = torch.zeros((R, K, C, D), device=DEV), rand((R, K, C, D), 1, torch.float32)
    x[:, :, where] = -below / (D * D ** -0.5)
    ck, clean = records(sv, x), records(sv, y)
    y[:, 1, where, 20:24] = torch.nan  # dimensions 16..31
    cv = records(sv, y)
    for window in (0, 40):
        want, tol, _, _ = attention(q, decode(ck, D), decode(clean, D), None, None, window, 2)
        got = sv.quantized_attention(q, ck, cv, window=window, sinks=2)
        assert torch.isnan(got[:, -2:, 2:, 16:32]).all()
        nan = torch.zeros_like(got, dtype=torch.bool)
        nan[:, -2:, 2:, 16:32] = True
        check(got[~nan], want[~nan], tol[~nan], "the rest")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,n,H,K,D", [(150, 1, 4, 2, 64), (40, 1, 36, 4, 128), (20, 5, 16, 2, 64), (1, 1, 8, 1, 128),
                                       (2, 100, 4, 2, 64), (1, 100, 9, 1, 128)])
@pytest.mark.parametrize("below", [20.5, 24.5, 25.2])
def test_many_light_slots_beside_a_heavy_one(sv, dtype, R, n, H, K, D, below):
    """A first slot of value zero that outweighs each other slot by 2^below: the others' share is the output.  A
    weight is held to 2^-32 of the heaviest (the 16-bit calls' operands: 2^-25 of what stands at 2^7), the rest is relative:
    the weights' and the values' roundings, the output's, 2^-18 for scores of 25, and half a step of 1 for each of the
    C / 4 weights at most that one thread adds to the heavy one."""
    C = 16384 if R < 100 else 8192
    x, y = torch.zeros((R, K, C, D), device=DEV, dtype=torch.float16), torch.ones((R, K, C, D), device=DEV, dtype=torch.float16)
    x[:, :, 0], y[:, :, 0] = 1.0, 0.0
    ck, cv = records(sv, x), records(sv, y)
    q = torch.ones((R, n, H, D), dtype=dtype, device=DEV)
    got = sv.quantized_attention(q, ck, cv, scale=below * math.log(2) / D)
    light = torch.arange(C - n, C, dtype=torch.float64, device=DEV)
    mass = light * 2.0 ** -below
    want = (mass / (1 + mass))[None, :, None, None].expand_as(got)
    relative = U[dtype] + 2.0 ** -18 + C / 4 * 2.0 ** -24 + (2 * 2.0 ** -11 if dtype != torch.float32 else 0.0)
    tol = relative * want + (light * 2.0 ** -32 + 2.0 ** -25 if dtype != torch.float32 else light * 0)[None, :, None, None]
    check(got, want, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 4, 90])
@pytest.mark.parametrize("up", [90, 100, 108, 113])
def test_large_queries_under_a_small_scale(sv, dtype, n, up):
    """Queries times 2^up under a scale times 2^-up are the same call."""
    R, H, K, D, C = 2, 8, 2, 128, 500
    q = rand((R, n, H, D), 2, dtype)
    ck, cv = records(sv, rand((R, K, C, D), 3, dtype)), records(sv, rand((R, K, C, D), 4, dtype))
    got = sv.quantized_attention(q * 2.0 ** up, ck, cv, scale=D ** -0.5 * 2.0 ** -up)
    assert torch.equal(got, sv.quantized_attention(q, ck, cv, scale=D ** -0.5))


@pytest.mark.parametrize("n", [1, 4, 90])
def test_a_scale_of_zero_under_large_queries(sv, n):
    """All slots weigh alike whatever the queries' size; a negative scale below float's range is as good as zero."""
    R, H, K, D, C = 2, 8, 2, 128, 300
    q = (rand((R, n, H, D), 2, torch.float32) * 2.0 ** 120).bfloat16()
    ck, cv = records(sv, rand((R, K, C, D), 3, torch.float32)), records(sv, rand((R, K, C, D), 4, torch.float32))
    want = sv.quantized_attention(torch.zeros_like(q), ck, cv)
    assert torch.equal(sv.quantized_attention(q, ck, cv, scale=0.0), want)
    assert torch.equal(sv.quantized_attention(rand(q.shape, 5, q.dtype), ck, cv, scale=-1e-60), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 90])
def test_window_attention_of_large_queries_under_a_small_scale(sv, dtype, n):
    """Over a 16- or 32-bit cache too: queries and keys times powers of two under a scale that takes them back."""
    R, H, K, D, C, up = 2, 8, 2, 64, 300, 0 if dtype == torch.float16 else 53
    q, k, v = rand((R, n, H, D), 6, dtype), rand((R, K, C, D), 7, dtype), rand((R, K, C, D), 8, dtype)
    got = sv.window_attention(q * 2.0 ** up, k * 2.0 ** up, v, scale=-0.125 * 4.0 ** -up)
    assert torch.equal(got, sv.window_attention(q, k, v, scale=-0.125))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,K,D", [(1, 4, 1, 128), (1, 16, 1, 96), (1, 9, 1, 64), (4, 8, 2, 128)])
def test_scores_are_exact(sv, dtype, n, H, K, D):
    """The weights (float32) of keys with middles up to 100 that cancel in the scores, under queries with one large
    value a group and many 2^-10 of it: the groups' sums have to be exact.  The bound: 2^-20 of sum |q k| per score,
    twice."""
    R, C, G = 2, 400, 32 if D > 64 else 16
    g = torch.Generator(device=DEV).manual_seed(5)
    q = ((torch.rand((R, n, H, D), generator=g, device=DEV) * 2 - 1) * 2.0 ** -10).to(dtype)
    q[..., ::G] = 1.0
    a = (torch.rand((R, K, C, 1), generator=g, device=DEV) * 200 - 100)
    x = torch.zeros((R, K, C, D), device=DEV)
    x[..., :G], x[..., G:2 * G] = a, -a
    x = x.half()
    ck, cv = records(sv, x), records(sv, rand((R, K, C, D), 6, torch.float16))
    assert torch.equal(decode(ck, D), x.double())
    w = torch.zeros((R, K, C), device=DEV)
    sv.quantized_attention(q, ck, cv, scale=1.0, weights=w)
    _, _, want, _ = attention(q, x.double(), decode(cv, D), scale=1.0)
    S = 2 * 100 * (1 + G * 2.0 ** -10)
    check(w, want, want * (math.expm1(2 * 2.0 ** -20 * S) + 2.0 ** -19) + 1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 4, 12, 90])
@pytest.mark.parametrize("size", [1000.0, 8000.0, 32000.0])
@pytest.mark.parametrize("quantized", [True, False])
def test_scores_far_past_the_whole_numbers_of_f32(sv, quantized, dtype, n, size):
    """Scores of +-2^30 and more, of which one is the whole softmax (rows of one slot and of none among them).  Two
    roundings: the weight's (and over records the value's) to float16 or the 16-bit cache's type, and the output's."""
    R, H, K, D, C = 2, 8, 2, 128, 60 if n != 12 else 12
    q = (rand((R, n, H, D), 7, torch.float32) * size).clamp(-60000, 60000).to(dtype)
    ck = records(sv, (rand((R, K, C, D), 8, torch.float32) * size).clamp(-30000, 30000))
    cv = records(sv, rand((R, K, C, D), 9, torch.float32))
    k, v = decode(ck, D), decode(cv, D)
    if quantized:
        got = sv.quantized_attention(q, ck, cv)
    else:
        k, v = k.to(dtype), v.to(dtype)
        got = sv.window_attention(q, k, v)
        k, v = k.double(), v.double()
    for r in range(R):
        for i in range(n):
            end = C - n + i + 1
            if end < 1:
                assert (got[r, i] == 0).all()
                continue
            s = q[r, i].double().view(K, H // K, D) @ k[r, :, :end].transpose(1, 2) * D ** -0.5
            S = q[r, i].double().abs().view(K, H // K, D) @ k[r, :, :end].abs().transpose(1, 2) * D ** -0.5
            top = s.topk(min(2, end), -1)
            # The others are behind by more than twice the scores' own error.
            clear = (top.values[..., 0] - top.values[..., -1] > 2.0 ** -9 * S.amax(-1) + 50) | (end == 1)
            want = torch.stack([v[r, h][top.indices[h, :, 0]] for h in range(K)]).view(H, D)
            off = (got[r, i].double() - want).abs()
            ok = off <= (U[dtype] + (2 * 2.0 ** -11 if quantized else U[dtype])) * want.abs() + 2.0 ** -24
            assert torch.isfinite(got[r, i]).all()
            assert ok.view(K, H // K, D)[clear].all()


def two_keys(sv, D, fine):
    """Records of two keys that stand for 1 +- a little: what lies below the last place of float16 at 1 (fine), or below
    bfloat16's only; and by how much their sums over the dimensions differ."""
    G = 32 if D > 64 else 16
    x = torch.ones((1, 1, 2, D), dtype=torch.float64, device=DEV)
    if fine:
        s = 2.0 ** -14
        x[:, :, 0], x[:, :, 1] = 1 + 7 * s, 1 - 8 * s
        x[:, :, 0, ::G], x[:, :, 1, ::G] = 1 - 8 * s, 1 + 7 * s
    else:
        x[:, :, 0] = 1 + 3 * 2.0 ** -10
    c = records(sv, x.float())
    assert torch.equal(decode(c, D), x)
    return c, (x[0, 0, 0].sum() - x[0, 0, 1].sum()).item()


def alternating(sv, dtype, R, n, H, K, D, C, fine=True):
    """Every second slot of half the weight's logarithm more: (q, scale, keys, values, shares [n], weights [n, C],
    relative bound).  What the rounded keys would do instead: weigh all alike, a share of 0.5 for 0.62."""
    two, apart = two_keys(sv, D, fine)
    ck = two.expand(R, K, 2, two.shape[-1]).repeat(1, 1, C // 2, 1)
    v = torch.zeros((1, 1, 2, D), device=DEV)
    v[:, :, 0] = 1.0
    cv = records(sv, v).expand(R, K, 2, two.shape[-1]).repeat(1, 1, C // 2, 1)
    q = torch.full((R, n, H, D), 2.0, dtype=dtype, device=DEV)
    scale = 0.25 / apart
    j = torch.arange(C, device=DEV)
    see = j <= torch.arange(C - n, C, device=DEV)[:, None]
    e = torch.where(see, torch.where(j % 2 == 0, math.exp(0.5), 1.0).double(), 0.0)
    p = e / e.sum(1, keepdim=True)
    share = p[:, ::2].sum(1)
    # Scores to 2^-20 of sum |q k| (about 2 D scale), twice; f32 sums of the slots that one thread adds.
    bound = math.expm1(2 * 2.0 ** -20 * 2 * D * scale) + C / 4 * 2.0 ** -24 + 2.0 ** -18
    return q, scale, ck, cv, share, p.sum(0), bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,n,H,K,D,C", [(40, 1, 36, 4, 128, 49152), (3, 5, 36, 4, 64, 131072), (1, 8, 32, 8, 64, 300000)])
def test_more_scores_than_are_kept(sv, dtype, R, n, H, K, D, C):
    """Accumulated weights of few query rows whose scores take more than 256 MB: cache rows, and heads of one row, in
    turn, with keys as exact as below that."""
    assert R * n * H * C * 4 > 1 << 28
    q, scale, ck, cv, share, weights, bound = alternating(sv, dtype, R, n, H, K, D, C)
    w = torch.zeros((R, K, C), device=DEV)
    status = i32([-1] * R)
    got = sv.quantized_attention(q, ck, cv, scale=scale, weights=w, status=status)
    assert status.tolist() == [0] * R
    roundings = U[dtype] + (2 * 2.0 ** -11 if dtype != torch.float32 else 0.0)
    want = share[None, :, None, None].expand_as(got)
    check(got, want, want * (bound + roundings))
    check(w, (H // K * weights).expand_as(w), (H // K * weights * bound).expand_as(w), "weights")
    # Other cache rows' queries and records reach a row: each on its own place.
    if R > 1:
        q[1], ck[1, 1:] = 0, ck[1, 1:].flip(1)
        w.zero_()
        again = sv.quantized_attention(q, ck, cv, scale=scale, weights=w)
        assert torch.equal(again[0], got[0]) and torch.equal(again[2:], got[2:])
        half = torch.arange(C - n + 1, C + 1, device=DEV)
        half = ((half + 1) // 2 / half.double())[:, None, None].expand_as(again[1])
        check(again[1], half, half * (bound + roundings), "a row of its own")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,n,H,K,D,C", [(2, 90, 8, 2, 64, 700), (1, 200, 16, 1, 128, 2000), (20, 70, 4, 4, 96, 20000),
                                         (3, 33, 36, 4, 128, 34)])
def test_weights_of_many_query_rows(sv, dtype, R, n, H, K, D, C):
    """Accumulated weights change nothing of the outputs, and are those of keys that the inputs' type does not hold."""
    q, scale, ck, cv, share, weights, bound = alternating(sv, dtype, R, n, H, K, D, C, fine=dtype != torch.bfloat16)
    plain = sv.quantized_attention(q, ck, cv, scale=scale)
    w = torch.zeros((R, K, C), device=DEV)
    got = sv.quantized_attention(q, ck, cv, scale=scale, weights=w)
    want = share[None, :, None, None].expand_as(got)
    roundings = U[dtype] + (2 * 2.0 ** -11 if dtype != torch.float32 else 0.0)
    check(plain, want, want * (bound + roundings))
    check(got, want, want * (bound + roundings))
    check(w, (H // K * weights).expand_as(w), (H // K * weights * bound).expand_as(w), "weights")
