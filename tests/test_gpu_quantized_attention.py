"""quantized_attention against attention in 64 bits over what the records stand for: types,
head layouts, lengths from one slot up, odd sizes, strides, rows that see nothing,
groups that stand for NaN in hidden slots, accumulated weights, streams and graphs.
Bounds: see _records_ref."""
import pytest
import torch

from _attention_ref import check
from _records_ref import attention, decode, record

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def cache(sv, shape, seed, dtype=torch.float16, scale=1.0, shift=0.0):
    """Random records [R, K, C, record(D)] of values scale * normal + shift."""
    c = torch.zeros(shape[:-1] + (record(shape[-1]),), dtype=torch.uint8, device=DEV)
    sv.kv_quantize(rand(shape, seed, dtype, scale) + shift, None, c, None)
    return c


# rows, tokens, heads, kv_heads, head_dim, capacity, window, sinks
TOKEN = [(1, 1, 1, 1, 64, 1, 0, 0), (2, 1, 16, 1, 128, 1000, 0, 0), (3, 1, 36, 4, 128, 517, 100, 4),
         (5, 1, 4, 4, 80, 333, 64, 1), (2, 1, 12, 2, 8, 77, 0, 0), (2, 1, 40, 1, 128, 300, 130, 7),
         (1, 1, 9, 1, 96, 5000, 4096, 64), (70, 1, 8, 8, 64, 130, 16, 16), (2, 3, 10, 2, 128, 700, 256, 4),
         (3, 16, 2, 2, 120, 65, 9, 2), (2, 1, 8, 1, 32, 900, 0, 0), (1, 1, 4, 1, 40, 100, 7, 1),
         (2, 5, 36, 4, 128, 1030, 0, 0), (1, 8, 8, 2, 64, 600, 64, 4), (300, 1, 1, 1, 128, 20, 0, 0)]
PROMPT = [(1, 2, 40, 1, 64, 2, 0, 0), (2, 65, 16, 1, 128, 65, 0, 0), (1, 300, 9, 1, 128, 300, 100, 4),
          (2, 129, 6, 3, 80, 500, 64, 1), (1, 577, 8, 2, 64, 600, 256, 300), (3, 33, 36, 4, 128, 190, 1, 0),
          (1, 257, 4, 4, 128, 1300, 0, 0), (2, 128, 4, 4, 128, 128, 128, 1), (1, 1000, 2, 1, 16, 1000, 333, 5),
          (1, 700, 1, 1, 128, 700, 0, 0), (2, 100, 8, 4, 96, 2100, 0, 0)]


def lengths_for(rows, n, capacity):
    step = max(1, (capacity - min(n, capacity)) // max(1, rows - 1))
    return [capacity - step * r if capacity - step * r >= n else n for r in range(rows)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TOKEN + PROMPT)
def test_quantized_attention(sv, shape, dtype):
    R, n, H, K, D, C, window, sinks = shape
    q = rand((R, n, H, D), 1, dtype, 1.5)
    ck, cv = cache(sv, (R, K, C, D), 2, shift=0.3), cache(sv, (R, K, C, D), 3)
    k, v = decode(ck, D), decode(cv, D)
    for lengths in (None, i32(lengths_for(R, n, C))):
        got = sv.quantized_attention(q, ck, cv, lengths, window=window, sinks=sinks)
        want, tol, _, _ = attention(q, k, v, lengths, None, window, sinks)
        assert got.dtype == dtype and got.shape == q.shape
        check(got, want, tol, f"{shape} {lengths}")
        again = sv.quantized_attention(q, ck, cv, lengths, window=window, sinks=sinks)
        assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 3, 7, 200])
def test_rows_that_see_nothing_and_padding(sv, dtype, n):
    """Lengths of zero and below the queries' count, starts that hide everything, and records of
    any bytes in every slot that no query sees."""
    R, H, K, D, C = 6, 8, 2, 128, 401
    q = rand((R, n, H, D), 4, dtype)
    lengths, starts = i32([0, 1, C, 150, 300, 300]), i32([0, 0, 17, 149, 300, 120])
    for window, sinks in ((0, 0), (50, 3), (1, 0)):
        ck, cv = cache(sv, (R, K, C, D), 5), cache(sv, (R, K, C, D), 6)
        k, v = decode(ck, D), decode(cv, D)
        for r in range(R):
            end, start = int(lengths[r]), int(starts[r])
            hidden = torch.ones(C, dtype=torch.bool, device=DEV)
            for p in range(max(start, end - n), end):
                lo = max(start, p - window + 1) if window else start
                hidden[lo:p + 1] = False
                hidden[start:min(start + sinks, p + 1)] = False
            ck[r, :, hidden] = 255
            cv[r, :, hidden] = (0x7c, 255)[r % 2]
        status = i32([-1] * R)
        got = sv.quantized_attention(q, ck, cv, lengths, starts=starts, window=window, sinks=sinks, status=status)
        want, tol, _, _ = attention(q, k, v, lengths, starts, window, sinks)
        check(got, want, tol, f"window {window}")
        assert (got[0] == 0).all() and (got[4] == 0).all()
        assert status.tolist() == [0] * R


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [3, 6, 64, 300])
def test_hidden_slots_reach_no_earlier_query(sv, dtype, n):
    """Groups that stand for NaN reach the queries that see their slot, and no others."""
    R, H, K, D, C = 1, 4, 2, 64, 320
    q = rand((R, n, H, D), 7, dtype)
    x, y = rand((R, K, C, D), 8, torch.float16), rand((R, K, C, D), 9, torch.float16)
    where = C - 2  # seen by the last two queries
    x2, y2 = x.clone(), y.clone()
    y2[:, 1, where, 20:24] = torch.inf   # dimensions 16..31 of values, head 1
    x2[:, 0, where, 3] = torch.nan       # keys, head 0
    ck, cv, ck2, cv2 = (torch.zeros((R, K, C, record(D)), dtype=torch.uint8, device=DEV) for _ in range(4))
    sv.kv_quantize(x, y, ck, cv)
    sv.kv_quantize(x2, y2, ck2, cv2)
    for window in (0, 40):
        plain = sv.quantized_attention(q, ck, cv, window=window, sinks=2)
        got = sv.quantized_attention(q, ck2, cv2, window=window, sinks=2)
        want, tol, _, _ = attention(q, decode(ck, D), decode(cv, D), None, None, window, 2)
        check(plain, want, tol)
        check(got[:, :-2], want[:, :-2], tol[:, :-2], "queries that do not see the slot")
        assert torch.isnan(got[:, -2:, :2]).all(), "a key that stands for NaN"
        assert torch.isnan(got[:, -2:, 2:, 16:32]).all(), "values that stand for NaN"
        rest = [d for d in range(D) if not 16 <= d < 32]
        check(got[:, -2:, 2:][..., rest], want[:, -2:, 2:][..., rest], tol[:, -2:, 2:][..., rest], "other dimensions")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,K,D,C,window", [(1, 16, 1, 128, 900, 0), (1, 36, 4, 128, 517, 100), (4, 8, 2, 64, 300, 0),
                                              (90, 8, 2, 64, 300, 70), (64, 16, 1, 128, 700, 0)])
def test_accumulated_weights(sv, dtype, n, H, K, D, C, window):
    R = 2
    q = rand((R, n, H, D), 10, dtype)
    ck, cv = cache(sv, (R, K, C, D), 11), cache(sv, (R, K, C, D), 12)
    lengths = i32([C, max(n, C - 37)])
    before = torch.rand((R, K, C), device=DEV)
    w = before.clone()
    got = sv.quantized_attention(q, ck, cv, lengths, window=window, sinks=4, weights=w)
    want, tol, wts, wtol = attention(q, decode(ck, D), decode(cv, D), lengths, None, window, 4)
    check(got, want, tol)
    total = before.double() + wts
    check(w, total, wtol + 2.0 ** -22 * total, "weights")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 50])
def test_layouts(sv, dtype, n):
    """Slots outside heads with gaps, broadcast heads, MQA forms, unaligned queries, a given output and scale."""
    R, H, K, D, C = 3, 12, 3, 128, 200
    wide = torch.zeros((R, C, 2, K, record(D) + 32), dtype=torch.uint8, device=DEV)
    ck, cv = (wide[:, :, i, :, :record(D)].transpose(1, 2) for i in range(2))
    sv.kv_quantize(rand((R, K, C, D), 13, dtype), rand((R, K, C, D), 14, dtype), ck, cv)
    q = rand((R * n * H * D + 1,), 15, dtype)[1:].view(R, n, H, D)
    k, v = decode(ck, D), decode(cv, D)
    lengths = i32([C, 150, 77])
    out = torch.empty_like(q)
    got = sv.quantized_attention(q, ck, cv, lengths, scale=-0.2, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, tol, _, _ = attention(q, k, v, lengths, scale=-0.2)
    check(got, want, tol, "gaps")
    dense = sv.quantized_attention(q, ck.contiguous(), cv.contiguous(), lengths, scale=-0.2)
    assert torch.equal(dense, got)
    one_k, one_v = (c[:1, :1].contiguous().expand(R, K, C, record(D)) for c in (ck, cv))
    got = sv.quantized_attention(q, one_k, one_v, lengths)
    want, tol, _, _ = attention(q, decode(one_k, D), decode(one_v, D), lengths)
    check(got, want, tol, "broadcast")
    got = sv.quantized_attention(q[:, :, :4], ck[:, 1], cv[:, 1], 130)
    want, tol, _, _ = attention(q[:, :, :4], k[:, 1:2, :130], v[:, 1:2, :130])
    check(got, want, tol, "MQA")
    if n == 1:
        three = sv.quantized_attention(q[:, 0], ck, cv, lengths)
        assert three.shape == (R, H, D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 4, 40])
def test_extreme_scores_and_scales(sv, dtype, n):
    """Scores far apart (a late maximum), keys far from zero, tiny and large groups, queries of
    very different sizes."""
    R, H, K, D, C = 2, 8, 2, 128, 700
    q = rand((R, n, H, D), 16, dtype)
    q[:, :, 1] *= 8
    q[:, :, 2] *= 1e-3
    q[:, :, 3] = 0
    x = rand((R, K, C, D), 17, torch.float32) + 4
    x[:, :, 600:610] *= 3
    x[:, :, 100:120] *= 1e-3
    y = rand((R, K, C, D), 18, torch.float32)
    y[:, :, ::7] *= 30
    y[:, :, 3::7] *= 1e-3
    ck, cv = (torch.zeros((R, K, C, record(D)), dtype=torch.uint8, device=DEV) for _ in range(2))
    sv.kv_quantize(x, y, ck, cv)
    got = sv.quantized_attention(q, ck, cv)
    want, tol, _, _ = attention(q, decode(ck, D), decode(cv, D))
    check(got, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_scale_of_zero_and_queries_that_are_not_finite(sv, dtype, n):
    """A scale of zero weighs all slots alike; a query with NaN makes its own row NaN, no others."""
    R, H, K, D, C = 2, 18, 2, 128, 333
    q = rand((R, n, H, D), 27, dtype)
    ck, cv = cache(sv, (R, K, C, D), 28), cache(sv, (R, K, C, D), 29)
    lengths = i32([C, max(n, 100)])
    k, v = decode(ck, D), decode(cv, D)
    got = sv.quantized_attention(q, ck, cv, lengths, scale=0.0, window=200, sinks=2)
    want, tol, _, _ = attention(q, k, v, lengths, None, 200, 2, 0.0)
    check(got, want, tol, "zero")
    q[:, n - 1, 3, 5] = torch.nan
    want, tol, _, _ = attention(q.nan_to_num(0.0), k, v, lengths)
    got = sv.quantized_attention(q, ck, cv, lengths)
    assert torch.isnan(got[:, n - 1, 3]).all()
    rest = torch.ones((n, H), dtype=torch.bool, device=DEV)
    rest[n - 1, 3] = False
    check(got[:, rest], want[:, rest], tol[:, rest], "others")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_many_rows_in_batches(sv, dtype, D):
    """More cache rows than are turned into plain values at a time, and two at the end."""
    R, n, H, K, C = 14, 70, 2, 2, 20000 if D == 128 else 40000
    q = rand((R, n, H, D), 30, dtype)
    ck, cv = cache(sv, (R, K, C, D), 31), cache(sv, (R, K, C, D), 32)
    lengths = i32([C - 911 * r for r in range(R)])
    status = i32([-1] * R)
    got = sv.quantized_attention(q, ck, cv, lengths, window=300, sinks=4, status=status)
    assert status.tolist() == [0] * R
    for r in (0, 1, 6, R - 2, R - 1):
        end = int(lengths[r])
        k, v = decode(ck[r:r + 1, :, :end], D), decode(cv[r:r + 1, :, :end], D)
        want, tol, _, _ = attention(q[r:r + 1], k, v, None, None, 300, 4)
        check(got[r:r + 1], want, tol, f"row {r}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_units_and_many(sv, dtype):
    """One unit in more parts than one block joins, and far more units than blocks."""
    for R, H, K, D, C in ((1, 8, 1, 128, 40000), (1, 16, 1, 64, 70000), (90, 9, 3, 128, 700)):
        q = rand((R, 1, H, D), 33, dtype)
        ck, cv = cache(sv, (R, K, C, D), 34), cache(sv, (R, K, C, D), 35)
        lengths = i32([max(1, C - 7 * r) for r in range(R)])
        got = sv.quantized_attention(q, ck, cv, lengths)
        want, tol, _, _ = attention(q, decode(ck, D), decode(cv, D), lengths)
        check(got, want, tol, f"{R} rows")
        assert torch.equal(got, sv.quantized_attention(q, ck, cv, lengths))


def test_streams_and_graphs(sv):
    R, H, K, D, C = 4, 36, 4, 128, 600
    q = rand((R, 1, H, D), 19, torch.bfloat16)
    ck, cv = cache(sv, (R, K, C, D), 20), cache(sv, (R, K, C, D), 21)
    lengths = i32([C, 300, 17, 1])
    want = sv.quantized_attention(q, ck, cv, lengths)
    long_q = rand((R, 90, H, D), 22, torch.bfloat16)
    want_long = sv.quantized_attention(long_q, ck, cv, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a = sv.quantized_attention(q, ck, cv, lengths)
            b = sv.quantized_attention(long_q, ck, cv, lengths)
        graphs.append((graph, a, b))
    with torch.cuda.stream(side):
        eager = sv.quantized_attention(q, ck, cv, lengths)
    other = torch.cuda.Stream()
    for _ in range(3):
        for graph, a, b in graphs:
            a.zero_()
            b.zero_()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for graph, a, b in graphs:
            assert torch.equal(a, want) and torch.equal(b, want_long)
    assert torch.equal(eager, want)


# Tokens, heads and key/value heads: single tokens, a draft in several groups of rows, and chunks past 64 rows.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,K", [(1, 36, 4), (1, 4, 4), (5, 36, 4), (40, 8, 2), (90, 36, 4)])
def test_output_in_the_queries_place(sv, dtype, n, H, K):
    """Outputs may take their own queries' place: many blocks share a unit (long rows) or blocks take many."""
    for R, C in ((2, 6000), (40, 300)):
        q = rand((R, n, H, 128), 40, dtype)
        ck, cv = cache(sv, (R, K, C, 128), 41), cache(sv, (R, K, C, 128), 42)
        lengths = i32(lengths_for(R, n, C))
        want = sv.quantized_attention(q, ck, cv, lengths, window=C // 2, sinks=3)
        for _ in range(3):
            x = q.clone()
            got = sv.quantized_attention(x, ck, cv, lengths, window=C // 2, sinks=3, out=x)
            assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)


def test_calls_that_share_a_kept_workspace(sv):
    """Calls of many sizes, types and kinds in turn on one stream give what each gives first: workspaces are kept by the
    power of two of their size, and plain and 4-bit calls share them."""
    calls = []
    for i, (R, n, H, K, D, C, dtype) in enumerate([
            (1, 1, 4, 1, 64, 40, torch.float16), (8, 1, 36, 4, 128, 3000, torch.bfloat16), (2, 90, 8, 2, 64, 700, torch.float16),
            (600, 1, 8, 8, 64, 60, torch.bfloat16), (3, 5, 36, 4, 128, 900, torch.float32), (2, 50, 36, 4, 128, 300, torch.float32),
            (4, 130, 36, 4, 128, 500, torch.bfloat16)]):
        q, ck, cv = rand((R, n, H, D), 50 + i, dtype), cache(sv, (R, K, C, D), 60 + i), cache(sv, (R, K, C, D), 70 + i)
        k, v = sv.kv_dequantize(ck, cv, D, dtype=dtype)
        calls.append(lambda q=q, ck=ck, cv=cv: sv.quantized_attention(q, ck, cv))
        calls.append(lambda q=q, k=k, v=v: sv.window_attention(q, k, v))
        calls.append(lambda q=q, ck=ck, cv=cv, R=R, K=K, C=C: sv.quantized_attention(
            q, ck, cv, weights=torch.zeros((R, K, C), device=DEV)))
    want = [call() for call in calls]
    for order in (range(len(calls)), reversed(range(len(calls))), [5 * i % len(calls) for i in range(len(calls))]):
        for i in order:
            assert torch.equal(calls[i](), want[i]), i


def test_decode_loop(sv):
    """A few steps as a decoder takes them: write the token, attend, reorder, evict; against 64 bits."""
    L, R, H, K, D, C = 1, 3, 8, 2, 64, 40
    ck = torch.zeros((L, R, K, C, record(D)), dtype=torch.uint8, device=DEV)
    cv = torch.zeros_like(ck)
    weights = torch.zeros((L, R, K, C), device=DEV)
    positions = torch.arange(C, dtype=torch.int32, device=DEV).expand(L, R, K, C).contiguous()
    lengths = i32([30, 22, 11])
    sv.kv_quantize(rand((R, K, 30, D), 23, torch.bfloat16), rand((R, K, 30, D), 24, torch.bfloat16), ck[0], cv[0], lengths)
    for step in range(12):
        lengths += 1
        sv.kv_quantize(rand((R, K, 1, D), 30 + step, torch.bfloat16), rand((R, K, 1, D), 60 + step, torch.bfloat16),
                       ck[0], cv[0], lengths)
        q = rand((R, 1, H, D), 90 + step, torch.bfloat16)
        got = sv.quantized_attention(q, ck[0], cv[0], lengths, weights=weights[0])
        want, tol, _, _ = attention(q, decode(ck[0], D), decode(cv[0], D), lengths)
        check(got, want, tol, f"step {step}")
        if step == 5:
            sv.kv_reorder(ck, cv, torch.tensor([1, 1, 0], device=DEV), C)
            lengths = lengths[torch.tensor([1, 1, 0], device=DEV)]
        if step == 8:
            cut = sv.kv_evict(ck, cv, weights, positions, lengths, 20, sinks=2, recent=4)
            weights, positions, lengths = cut["weights"], cut["positions"], cut["lengths"]


def test_empty(sv):
    q = rand((2, 1, 4, 64), 25, torch.float16)
    c = torch.zeros((2, 2, 0, record(64)), dtype=torch.uint8, device=DEV)
    status = i32([-1, -1])
    got = sv.quantized_attention(q, c, c.clone(), i32([0, 1]), status=status)
    assert (got == 0).all() and status.tolist() == [0, 8]
    c = cache(sv, (2, 2, 5, 64), 26)
    assert sv.quantized_attention(q[:, :0], c, c.clone()).shape == (2, 0, 4, 64)


def test_refusals(sv):
    q = torch.zeros((2, 1, 4, 128), device=DEV, dtype=torch.float16)
    c = torch.zeros((2, 2, 8, 80), device=DEV, dtype=torch.uint8)
    w = torch.zeros((2, 2, 8), device=DEV)
    for bad, error in [
            (lambda: sv.quantized_attention(q, c.half(), c.half()), ValueError),
            (lambda: sv.quantized_attention(q, c[..., :64], c[..., :64]), ValueError),
            (lambda: sv.quantized_attention(q[..., :64], c, c), ValueError),
            (lambda: sv.quantized_attention(q[..., :100], c, c), ValueError),
            (lambda: sv.quantized_attention(q, c, c[:, :, :4]), ValueError),
            (lambda: sv.quantized_attention(q[:1], c, c), ValueError),
            (lambda: sv.quantized_attention(q[:, :, :3], c, c), ValueError),
            (lambda: sv.quantized_attention(q, c, c, 9), ValueError),
            (lambda: sv.quantized_attention(q, c, c, window=-1), ValueError),
            (lambda: sv.quantized_attention(q, c, c, scale=float("nan")), ValueError),
            (lambda: sv.quantized_attention(q, c, c, weights=w[:1].expand(2, 2, 8)), ValueError),
            (lambda: sv.quantized_attention(q, c, c, weights=w, out=q), RuntimeError),
            (lambda: sv.quantized_attention(q.cpu(), c, c), RuntimeError),
            (lambda: sv.quantized_attention(q, c.cpu(), c.cpu()), RuntimeError),
            (lambda: sv.quantized_attention(q, c[:, :, :1].expand(2, 2, 8, 80), c[:, :, :1].expand(2, 2, 8, 80)),
             RuntimeError),
            (lambda: sv.quantized_attention(q, c, c, status=torch.zeros((2, 2), dtype=torch.int32, device=DEV)[:, 0]),
             RuntimeError)]:
        with pytest.raises(error):
            bad()
