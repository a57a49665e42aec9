"""kv_quantize and kv_dequantize against the format in 64 bits: codes and pairs exactly,
at ties and next to them, constants, values that are not finite or past the range;
layouts, lengths, other slots untouched, streams and graphs; and records under
kv_reorder and kv_evict."""
import numpy as np
import pytest
import torch

from _records_ref import decode, encode, record, same_values

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DIMS = [128, 64, 80, 96, 32, 8, 40, 72, 120]


def rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def new_cache(R, K, C, D, fill=0):
    return torch.full((R, K, C, record(D)), fill, dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", DIMS)
def test_round_trip(sv, D, dtype):
    for R, K, n, C in ((1, 1, 1, 1), (2, 3, 5, 9), (3, 2, 70, 100), (1, 4, 33, 33), (5, 1, 2, 300)):
        k, v = rand((R, K, n, D), 1, dtype, 2.0), rand((R, K, n, D), 2, dtype) + 3
        ck, cv = new_cache(R, K, C, D, 7), new_cache(R, K, C, D, 9)
        lengths = i32([max(1, C - 3 * r) for r in range(R)])
        status = i32([-1] * R)
        assert sv.kv_record_bytes(D) == record(D)
        sv.kv_quantize(k, v, ck, cv, lengths, status=status)
        assert status.tolist() == [0] * R
        gk, gv = sv.kv_dequantize(ck, cv, D, lengths, tokens=n, dtype=dtype)
        for x, c, got, fill in ((k, ck, gk, 7), (v, cv, gv, 9)):
            want = new_cache(R, K, C, D, fill).cpu().numpy()
            back = torch.zeros((R, K, n, D), dtype=torch.float64)
            for r in range(R):
                end = int(lengths[r])
                m = min(n, end)
                want[r, :, end - m:end] = encode(x[r, :, n - m:].double().cpu().numpy())
                back[r, :, n - m:] = decode(torch.from_numpy(want[r, :, end - m:end]), D)
            assert same_values(c, want, D)
            off = (got.double().cpu() - back).abs()
            assert got.dtype == dtype and (off <= torch.finfo(dtype).eps / 2 * back.abs() * 1.001 + 2.0 ** -25).all()


@pytest.mark.parametrize("D", [128, 64])
def test_borders_between_codes(sv, D):
    """Values on and next to the borders of codes and of the float16 pairs, in float32."""
    g = np.random.default_rng(0)
    rows = []
    for _ in range(400):
        s = np.float16(2.0 ** g.integers(-12, 8) * (1 + g.integers(0, 1024) / 1024)).astype(np.float64)
        m = np.float16(g.standard_normal() * 2.0 ** g.integers(-6, 9)).astype(np.float64)
        x = m + s * (g.integers(0, 15, D) + 0.5 - 8)
        x[::32], x[1::32], x[16::32], x[17::32] = m - 8 * s, m + 7 * s, m - 8 * s, m + 7 * s
        x = x.astype(np.float32)
        up = g.integers(-1, 2, D)
        x = np.where(up > 0, np.nextafter(x, np.float32(np.inf)), np.where(up < 0, np.nextafter(x, np.float32(-np.inf)), x))
        rows.append(x)
        # Extremes whose fifteenth is a border of float16, or next to one.
        h = (1024 + g.integers(0, 1024) + 0.5) * 2.0 ** g.integers(-20, 2)
        y = np.full(D, 15 * h / 2, np.float32)
        y[::16] = np.nextafter(np.float32(-15 * h / 2), np.float32(g.choice([-np.inf, np.inf, -15 * h / 2])))
        rows.append(y)
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).to(DEV)[:, None, None]
    c = new_cache(x.shape[0], 1, 1, D)
    sv.kv_quantize(x, None, c, None)
    assert same_values(c, encode(x.double().cpu().numpy()), D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [128, 64, 40])
def test_odd_values(sv, D, dtype):
    """Constants, zeros of either sign, tiny and huge values, and what is not finite."""
    big = torch.finfo(dtype).max
    rows = [torch.zeros(D), torch.full((D,), -0.0), torch.full((D,), 1.2345), torch.full((D,), 1e-7),
            torch.linspace(-1, 1, D) * 1e-6, torch.linspace(-1, 1, D) * 2.0 ** -24, torch.linspace(-1, 1, D) * 40000.0,
            torch.linspace(20000, 60000, D), torch.linspace(-60000, -40000, D), 1000 + torch.linspace(-1, 1, D) * 1e-3,
            torch.where(torch.arange(D) % 7 == 0, big, -big * 0.5), 32768 + torch.linspace(-9, 9, D)]
    for bad in (torch.nan, torch.inf, -torch.inf):
        x = torch.linspace(-2, 3, D)
        x[5] = bad
        rows.append(x)
        rows.append(torch.full((D,), bad))
    x = torch.stack(rows).to(dtype).to(DEV)[:, None, None]
    c = new_cache(x.shape[0], 1, 1, D, 255)
    sv.kv_quantize(x, None, c, None)
    assert same_values(c, encode(x.double().cpu().numpy()), D)
    for out in DTYPES:
        got, none = sv.kv_dequantize(c, None, D, dtype=out)
        assert none is None
        want = decode(c, D)
        assert (torch.isnan(got) == torch.isnan(want)).all()
        off = (got.double() - want).abs().nan_to_num(0.0)
        assert (off <= torch.finfo(out).eps / 2 * want.abs().nan_to_num(0.0) * 1.001 + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(sv, dtype):
    """A fused projection in place, MQA forms, odd strides (copied), caches with gaps, slots outside heads."""
    R, n, K, D, C = 3, 21, 2, 128, 40
    x = rand((R, n, 7 * K * D), 3, dtype)
    k = x[..., 5 * K * D:6 * K * D].unflatten(2, (K, D)).transpose(1, 2)
    v = x[..., 6 * K * D:].unflatten(2, (K, D)).transpose(1, 2)
    want_k, want_v = (encode(t.double().cpu().numpy()) for t in (k, v))
    lengths = i32([40, 30, 21])

    def check(ck, cv, lens):
        for c, w in ((ck, want_k), (cv, want_v)):
            for r in range(R):
                assert same_values(c[r][:, int(lens[r]) - n:int(lens[r])], w[r], D)

    wide = torch.zeros((R, C, 2, K, record(D) + 16), dtype=torch.uint8, device=DEV)  # slots outside heads, gaps
    ck, cv = (wide[:, :, i, :, :record(D)].transpose(1, 2) for i in range(2))
    sv.kv_quantize(k, v, ck, cv, lengths)
    check(ck, cv, lengths)
    assert (wide[..., record(D):] == 0).all()
    for dt in DTYPES:
        a = sv.kv_dequantize(ck, cv, D, lengths, dtype=dt)
        b = sv.kv_dequantize(ck.contiguous(), cv.contiguous(), D, lengths, dtype=dt)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for r in range(R):
            assert (a[0][r, :, int(lengths[r]):] == 0).all()
    # Strides of their own, an offset of one element, a broadcast head.
    odd = rand((R * K * n * D + 1,), 4, dtype)[1:].view(R, K, n, D)
    one = rand((R, 1, n, D), 5, dtype).expand(R, K, n, D)
    ck, cv = new_cache(R, K, C, D), new_cache(R, K, C, D)
    sv.kv_quantize(odd, one, ck, cv)
    assert same_values(ck[:, :, C - n:], encode(odd.double().cpu().numpy()), D)
    assert same_values(cv[:, :, C - n:], encode(one.double().cpu().numpy()), D)
    # MQA without a head dimension, a number as length, int64 lengths.
    mk, mv = k[:, 0], v[:, 0]
    ck, cv = new_cache(R, 1, C, D)[:, 0], new_cache(R, 1, C, D)[:, 0]
    sv.kv_quantize(mk, mv, ck, cv, 25)
    assert same_values(ck[:, 4:25], want_k[:, 0], D) and (ck[:, 25:] == 0).all() and (ck[:, :4] == 0).all()
    got = sv.kv_dequantize(ck, cv, D, 25, tokens=n, dtype=dtype)
    assert got[0].shape == (R, n, D)
    whole = sv.kv_dequantize(ck, cv, D, torch.tensor([25] * R, device=DEV), dtype=dtype)
    assert torch.equal(whole[0][:, 4:25], got[0]) and whole[1].shape == (R, C, D)


def test_lengths(sv):
    """Rows with fewer slots than tokens, empty rows, lengths outside the cache (clamped, reported)."""
    R, K, n, C, D = 6, 2, 5, 12, 64
    k = rand((R, K, n, D), 6, torch.float16)
    lengths = i32([0, 2, 12, 13, -4, 5])
    ck = new_cache(R, K, C, D, 3)
    status = i32([-1] * R)
    sv.kv_quantize(k, None, ck, None, lengths, status=status)
    assert status.tolist() == [0, 0, 0, 8, 8, 0]
    want = new_cache(R, K, C, D, 3).cpu().numpy()
    for r, end in enumerate([0, 2, 12, 12, 0, 5]):
        m = min(n, end)
        want[r, :, end - m:end] = encode(k[r, :, n - m:].double().cpu().numpy())
    assert np.array_equal(ck.cpu().numpy(), want)
    status = i32([-1] * R)
    got, _ = sv.kv_dequantize(ck, None, D, lengths, tokens=n, status=status)
    assert status.tolist() == [0, 0, 0, 8, 8, 0]
    assert (got[0] == 0).all() and (got[4] == 0).all() and (got[1, :, :3] == 0).all() and (got[1, :, 3:] != 0).any()
    # More places than slots.
    more, _ = sv.kv_dequantize(ck, None, D, lengths, tokens=20)
    assert (more[:, :, :8] == 0).all() and torch.equal(more[2, :, 15:], got[2])


def test_no_tokens(sv):
    ck = new_cache(2, 1, 8, 128)
    status = i32([-1, -1])
    sv.kv_quantize(torch.empty((2, 1, 0, 128), device=DEV), None, ck, None, i32([3, 9]), status=status)
    assert status.tolist() == [0, 8] and (ck == 0).all()
    k, v = sv.kv_dequantize(ck, ck.clone(), 128, tokens=0)
    assert k.shape == (2, 1, 0, 128) == v.shape


def test_reorder_and_evict_move_records(sv):
    """kv_reorder and kv_evict on uint8 caches, against the same on decoded values."""
    L, R, K, C, D = 2, 4, 2, 50, 128
    k, v = rand((L, R, K, C, D), 7, torch.float16), rand((L, R, K, C, D), 8, torch.float16)
    ck = torch.zeros((L, R, K, C, record(D)), dtype=torch.uint8, device=DEV)
    cv = torch.zeros_like(ck)
    for i in range(L):
        sv.kv_quantize(k[i], v[i], ck[i], cv[i])
    plain = [torch.stack([sv.kv_dequantize(ck[i], cv[i], D)[j] for i in range(L)]) for j in range(2)]
    parents = torch.tensor([2, 0, 2, 3], device=DEV)
    sv.kv_reorder(ck, cv, parents, 41)
    sv.kv_reorder(plain[0], plain[1], parents, 41)
    weights = torch.rand((L, R, K, C), device=DEV)
    positions = torch.arange(C, dtype=torch.int32, device=DEV).expand(L, R, K, C).contiguous()
    lengths = i32([41, 20, 33, 41])
    a = sv.kv_evict(ck, cv, weights, positions, lengths, 24, sinks=2, recent=5)
    b = sv.kv_evict(plain[0], plain[1], weights, positions, lengths, 24, sinks=2, recent=5)
    assert all(torch.equal(a[x], b[x]) for x in a)
    for i in range(L):
        got = sv.kv_dequantize(ck[i], cv[i], D)
        assert torch.equal(got[0], plain[0][i]) and torch.equal(got[1], plain[1][i])


def test_streams_and_graphs(sv):
    R, K, C, D = 3, 2, 64, 128
    ck, cv = new_cache(R, K, C, D), new_cache(R, K, C, D)
    k, v = rand((R, K, 1, D), 9, torch.bfloat16), rand((R, K, 1, D), 10, torch.bfloat16)
    lengths = i32([5, 6, 7])
    sv.kv_quantize(k, v, ck, cv, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        sv.kv_quantize(k, v, ck, cv, lengths)
        out = sv.kv_dequantize(ck, cv, D, lengths, tokens=3, dtype=torch.bfloat16)
        lengths += 1
    for step in range(3):
        k.copy_(rand((R, K, 1, D), 20 + step, torch.bfloat16))
        graph.replay()
        want = torch.from_numpy(encode(k.double().cpu().numpy()))
        for r in range(R):
            at = 4 + r + step
            assert same_values(ck[r, :, at:at + 1], want[r].numpy(), D)
            assert torch.equal(out[0][r, :, 2], decode(want[r, :, 0], D).to(DEV).to(torch.bfloat16))


def test_offsets_past_32_bits(sv):
    """Rows four gigabytes apart, the keys' and values' records interleaved."""
    C, D = 300, 128
    memory = torch.empty(((4 << 30) + 2 * C * record(D),), dtype=torch.uint8, device=DEV)
    ck, cv = (memory.as_strided((2, 1, C, record(D)), (4 << 30, 0, 2 * record(D), 1), i * record(D)) for i in range(2))
    k, v = rand((2, 1, C, D), 11, torch.bfloat16), rand((2, 1, C, D), 12, torch.bfloat16)
    sv.kv_quantize(k, v, ck, cv)
    a = sv.kv_dequantize(ck, cv, D)
    q = rand((2, 1, 9, D), 13, torch.bfloat16)
    b = sv.quantized_attention(q, ck, cv)
    many = rand((2, 40, 9, D), 14, torch.bfloat16)
    c = sv.quantized_attention(many, ck, cv)
    dense = [x.contiguous() for x in (ck, cv)]
    assert same_values(dense[0], encode(k.double().cpu().numpy()), D)
    assert same_values(dense[1], encode(v.double().cpu().numpy()), D)
    for got, want in zip(a, sv.kv_dequantize(*dense, D)):
        assert torch.equal(got, want)
    assert torch.equal(b, sv.quantized_attention(q, *dense)) and torch.equal(c, sv.quantized_attention(many, *dense))


def test_refusals(sv):
    k = torch.zeros((2, 1, 4, 128), device=DEV, dtype=torch.float16)
    ck, cv = new_cache(2, 1, 8, 128), new_cache(2, 1, 8, 128)
    for bad, error in [
            (lambda: sv.kv_record_bytes(100), ValueError),
            (lambda: sv.kv_quantize(k.to(torch.float64), None, ck, None), ValueError),
            (lambda: sv.kv_quantize(k, None, ck, cv), ValueError),
            (lambda: sv.kv_quantize(k, k[:, :, :3], ck, cv), ValueError),
            (lambda: sv.kv_quantize(k, None, ck[..., :64], None), ValueError),
            (lambda: sv.kv_quantize(k, None, ck.to(torch.int8), None), ValueError),
            (lambda: sv.kv_quantize(k[:1], None, ck, None), ValueError),
            (lambda: sv.kv_quantize(k, None, ck, None, 9), ValueError),
            (lambda: sv.kv_quantize(k, None, ck, None, 0), ValueError),
            (lambda: sv.kv_quantize(k, None, ck, None, i32([1, 2, 3])), ValueError),
            (lambda: sv.kv_quantize(k, k, ck, ck), RuntimeError),
            (lambda: sv.kv_quantize(k[:, :, :3], k[:, :, :3], ck[:, :, :7], ck[:, :, 1:]), RuntimeError),
            (lambda: sv.kv_quantize(k, None, ck[:1].expand(2, 1, 8, 80), None), RuntimeError),
            (lambda: sv.kv_quantize(k, None, ck[:, :, :1].expand(2, 1, 8, 80), None), RuntimeError),
            (lambda: sv.kv_quantize(k.cpu(), None, ck, None), RuntimeError),
            (lambda: sv.kv_quantize(k, None, ck.cpu(), None), RuntimeError),
            (lambda: sv.kv_dequantize(ck, cv, 64), ValueError),
            (lambda: sv.kv_dequantize(ck, cv, 128, tokens=-1), ValueError),
            (lambda: sv.kv_dequantize(ck, cv, 128, dtype=torch.float64), ValueError),
            (lambda: sv.kv_dequantize(ck, cv[:, :, :4], 128), ValueError),
            (lambda: sv.kv_dequantize(ck, None, 128, out=(torch.zeros(3, device=DEV), None)), RuntimeError),
            (lambda: sv.kv_dequantize(ck, cv, 128, out=(k.new_zeros((2, 1, 8, 128)),) * 2), RuntimeError)]:
        with pytest.raises(error):
            bad()
    assert (ck == 0).all() and (cv == 0).all()
