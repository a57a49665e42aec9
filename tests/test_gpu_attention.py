"""window_attention and prefix_attention against attention in 64 bits: types, head
layouts, lengths from one slot up, odd sizes, strides, rows that see nothing, garbage
in hidden slots, streams and graphs.  Bounds: see _attention_ref."""
import pytest
import torch

from _attention_ref import attention, check

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# rows, tokens, heads, kv_heads, head_dim, capacity, window, sinks
TOKEN = [(1, 1, 1, 1, 64, 1, 0, 0), (2, 1, 16, 1, 128, 1000, 0, 0), (3, 1, 36, 4, 128, 517, 100, 4),
         (5, 1, 4, 4, 80, 333, 64, 1), (2, 1, 12, 2, 8, 77, 0, 0), (2, 1, 40, 1, 128, 300, 130, 7),
         (1, 1, 9, 1, 96, 5000, 4096, 64), (70, 1, 8, 8, 64, 130, 16, 16), (2, 3, 10, 2, 128, 700, 256, 4),
         (3, 16, 2, 2, 120, 65, 9, 2)]
PROMPT = [(1, 2, 2, 1, 64, 2, 0, 0), (2, 65, 16, 1, 128, 65, 0, 0), (1, 300, 9, 1, 128, 300, 100, 4),
          (2, 129, 6, 3, 80, 500, 64, 1), (1, 577, 8, 2, 64, 600, 256, 300), (3, 33, 36, 4, 128, 190, 1, 0),
          (1, 257, 4, 4, 128, 1300, 0, 0), (2, 128, 4, 4, 128, 128, 128, 1), (1, 1000, 2, 1, 16, 1000, 333, 5),
          (1, 700, 1, 1, 128, 700, 0, 0)]


def lengths_for(rows, n, capacity):
    step = max(1, (capacity - min(n, capacity)) // max(1, rows - 1))
    return [capacity - step * r if capacity - step * r >= n else n for r in range(rows)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TOKEN + PROMPT)
def test_window_attention(sv, shape, dtype):
    R, n, H, K, D, C, window, sinks = shape
    q, k, v = rand((R, n, H, D), 1, dtype, 1.5), rand((R, K, C, D), 2, dtype), rand((R, K, C, D), 3, dtype)
    for lengths in (None, i32(lengths_for(R, n, C))):
        got = sv.window_attention(q, k, v, lengths, window=window, sinks=sinks)
        want, tol, _, _ = attention(q, k, v, lengths, None, window, sinks)
        assert got.dtype == dtype and got.shape == q.shape
        check(got, want, tol, f"{shape} {lengths}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 200])
def test_rows_that_see_nothing_and_padding(sv, dtype, n):
    """Lengths of zero and below the queries' count, starts that hide everything, and
    NaN / infinities in every slot that no query sees."""
    R, H, K, D, C = 6, 8, 2, 128, 401
    q, k, v = rand((R, n, H, D), 4, dtype), rand((R, K, C, D), 5, dtype), rand((R, K, C, D), 6, dtype)
    lengths, starts = i32([0, 1, C, 150, 300, 300]), i32([0, 0, 17, 149, 300, 120])
    for window, sinks in ((0, 0), (50, 3), (1, 0)):
        for r in range(R):
            end, start = int(lengths[r]), int(starts[r])
            hidden = torch.ones(C, dtype=torch.bool, device=DEV)
            for p in range(max(start, end - n), end):
                lo = max(start, p - window + 1) if window else start
                hidden[lo:p + 1] = False
                hidden[start:min(start + sinks, p + 1)] = False
            k[r, :, hidden] = torch.nan
            v[r, :, hidden] = torch.inf if r % 2 else torch.nan
        status = i32([-1] * R)
        got = sv.window_attention(q, k, v, lengths, starts=starts, window=window, sinks=sinks, status=status)
        want, tol, _, _ = attention(q, k, v, lengths, starts, window, sinks)
        check(got, want, tol, f"window {window}")
        assert (got[0] == 0).all() and (got[4] == 0).all()
        assert status.tolist() == [0] * R
        k, v = rand((R, K, C, D), 5, dtype), rand((R, K, C, D), 6, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [3, 64, 300])
def test_hidden_slots_reach_no_earlier_query(sv, dtype, n):
    """A NaN or infinity in a slot that only later (or only earlier) queries see stays
    out of the outputs of those that do not see it."""
    H, K, D, C, window = 4, 2, 64, 600, 70
    q, k, v = rand((1, n, H, D), 7, dtype), rand((1, K, C, D), 8, dtype), rand((1, K, C, D), 9, dtype)
    bad = C - n + n // 2  # the middle query's own slot
    clean = sv.window_attention(q, k, v, window=window)
    v[0, :, bad, 3] = torch.nan
    k[0, 1, bad] = torch.inf
    got = sv.window_attention(q, k, v, window=window)
    sees = torch.zeros(n, dtype=torch.bool)
    for i in range(n):
        p = C - n + i
        sees[i] = bad <= p and bad > p - window
    assert torch.equal(got[0, ~sees], clean[0, ~sees])
    assert torch.isnan(got[0, sees][..., 3]).all()
    finite = got[0, sees][:, :2, [d for d in range(D) if d != 3]]  # head group 0: only one dimension is bad
    assert torch.isfinite(finite).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_extreme_scores(sv, dtype, n):
    """Scores of +-hundreds: weights that underflow, a maximum that comes last, the
    lowest value of the type as a score's factor."""
    R, H, K, D, C = 2, 4, 1, 128, 450
    q, k, v = rand((R, n, H, D), 10, dtype, 6.0), rand((R, K, C, D), 11, dtype, 6.0), rand((R, K, C, D), 12, dtype)
    k[:, :, -1] = 3 * q[:, :1, 0, :].transpose(1, 2).reshape(R, 1, D).clamp(-40, 40)
    check(sv.window_attention(q, k, v), *attention(q, k, v)[:2], "large")
    k[:, :, 5] = torch.finfo(dtype).min  # a slot masked by its keys' lowest value
    q = q.abs()
    check(sv.window_attention(q, k, v, scale=0.01), *attention(q, k, v, scale=0.01)[:2], "lowest")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 90])
def test_strides_layouts_and_scale(sv, dtype, n):
    """Views: a fused projection read in place, a slot-major cache, an MQA cache without
    a head dimension, a broadcast row, an unaligned query, a preallocated output."""
    R, H, K, D = 3, 6, 2, 64
    x = rand((R, 200, (H + 2 * K) * D), 13, dtype)
    q = x[:, 200 - n:, :H * D].unflatten(2, (H, D))
    k = x[:, :, H * D:(H + K) * D].unflatten(2, (K, D)).transpose(1, 2)
    v = x[:, :, (H + K) * D:].unflatten(2, (K, D)).transpose(1, 2)
    check(sv.window_attention(q, k, v, window=33, sinks=2), *attention(q, k, v, None, None, 33, 2)[:2], "fused")
    out = torch.empty((R, n, H, D), dtype=dtype, device=DEV)
    assert sv.window_attention(q, k, v, 150, scale=0.3, out=out) is out
    check(out, *attention(q, k[:, :, :150], v[:, :, :150], scale=0.3)[:2], "number of slots, scale")
    mk, mv = k[:, 0], v[:, 0]
    check(sv.window_attention(q, mk, mv), *attention(q, mk[:, None], mv[:, None])[:2], "mqa")
    one = k[:1].expand(R, -1, -1, -1)
    two = v[:1].expand(R, -1, -1, -1)
    check(sv.window_attention(q, one, two), *attention(q, one, two)[:2], "broadcast rows")
    odd = rand((R * n * H * D + 1,), 14, dtype)[1:].view(R, n, H, D)
    check(sv.window_attention(odd, k, v), *attention(odd, k, v)[:2], "unaligned q")
    if n == 1:
        got = sv.window_attention(q[:, 0], k, v, torch.tensor([200, 9, 1]))
        assert got.shape == (R, H, D)
        check(got[:, None], *attention(q, k, v, [200, 9, 1])[:2], "three dimensions, host lengths")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 1, 0, 0), (3, 1, 36, 4, 128, 700, 0, 0), (2, 1, 16, 1, 80, 1200, 300, 4),
                                   (2, 5, 6, 2, 128, 333, 0, 0), (2, 150, 4, 2, 64, 300, 64, 2), (1, 1, 40, 2, 128, 90, 0, 0)])
def test_weights_accumulate(sv, shape, dtype):
    R, n, H, K, D, C, window, sinks = shape
    q, k, v = rand((R, n, H, D), 15, dtype, 1.5), rand((R, K, C, D), 16, dtype), rand((R, K, C, D), 17, dtype)
    lengths = i32(lengths_for(R, n, C))
    lengths[-1] = max(1, C // 3)
    before = torch.rand((R, K, C + 3), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    w = before.clone()
    got = sv.window_attention(q, k, v, lengths, window=window, sinks=sinks, weights=w)
    want, tol, wts, wtol = attention(q, k, v, lengths, None, window, sinks)
    check(got, want, tol, "out")
    check(w[:, :, :C], before[:, :, :C].double() + wts, wtol + 2.0 ** -23 * (before[:, :, :C] + wts) + 1e-30, "weights")
    assert torch.equal(w[:, :, C:], before[:, :, C:])
    for r in range(R):  # slots past the row's length keep their bits
        assert torch.equal(w[r, :, int(lengths[r]):], before[r, :, int(lengths[r]):])
    # Each query's weights sum to one.
    seen = torch.tensor([min(n, int(lengths[r])) for r in range(R)], device=DEV)
    total = (w.double() - before.double()).sum((1, 2))
    assert torch.allclose(total, seen.double() * H, rtol=1e-4, atol=1e-3)


# rows, tokens, heads, kv_heads, head_dim, prefix, capacity
PREFIX = [(1, 1, 1, 1, 64, 1, 1), (8, 1, 16, 1, 128, 1025, 100), (5, 1, 36, 4, 128, 333, 77), (33, 1, 8, 8, 64, 129, 50),
          (70, 1, 18, 2, 128, 700, 20), (3, 9, 8, 2, 80, 64, 40), (2, 130, 4, 2, 128, 500, 200), (4, 2, 6, 3, 8, 2000, 3),
          (6, 1, 40, 1, 128, 90, 300), (2, 1, 4, 2, 64, 0, 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", PREFIX)
def test_prefix_attention(sv, shape, dtype):
    R, n, H, K, D, P, C = shape
    q, k, v = rand((R, n, H, D), 18, dtype, 1.5), rand((R, K, C, D), 19, dtype), rand((R, K, C, D), 20, dtype)
    pk, pv = rand((K, P, D), 21, dtype), rand((K, P, D), 22, dtype)
    for lengths in (None, i32(lengths_for(R, n, C))):
        got = sv.prefix_attention(q, pk, pv, k, v, lengths)
        check(got, *attention(q, k, v, lengths, prefix=(pk, pv))[:2], f"{shape}")
    if P > 1:
        got = sv.prefix_attention(q, pk, pv, k, v, lengths, prefix_length=P - 1, scale=0.2)
        check(got, *attention(q, k, v, lengths, prefix=(pk[:, :-1], pv[:, :-1]), scale=0.2)[:2], "prefix_length")
        whole = torch.cat([pk[None].expand(R, -1, -1, -1), k], 2)
        both = torch.cat([pv[None].expand(R, -1, -1, -1), v], 2)
        got, same = sv.prefix_attention(q, pk, pv, k, v), sv.window_attention(q, whole, both)
        want, tol, _, _ = attention(q, whole, both)
        check(got, want, tol, "whole")
        check(same, want, tol, "as one cache")


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefix_rows_without_own_slots(sv, dtype):
    """Own lengths of zero: only the prefix is seen; garbage in unused slots stays out."""
    R, H, K, D, P, C = 3, 16, 1, 128, 200, 64
    q, k, v = rand((R, 1, H, D), 23, dtype), rand((R, C, D), 24, dtype), rand((R, C, D), 25, dtype)
    pk, pv = rand((P, D), 26, dtype), rand((P, D), 27, dtype)
    lengths = i32([0, 1, 40])
    for r in range(R):
        k[r, int(lengths[r]):], v[r, int(lengths[r]):] = torch.nan, torch.inf
    got = sv.prefix_attention(q, pk, pv, k, v, lengths)
    check(got, *attention(q, k[:, None], v[:, None], lengths, prefix=(pk[None], pv[None]))[:2])


def test_results_repeat_bit_for_bit(sv):
    """The joining order of the splits is fixed."""
    q, k, v = rand((4, 1, 36, 128), 28, torch.bfloat16), rand((4, 4, 3000, 128), 29, torch.bfloat16), \
        rand((4, 4, 3000, 128), 30, torch.bfloat16)
    pk, pv = rand((4, 900, 128), 31, torch.bfloat16), rand((4, 900, 128), 32, torch.bfloat16)
    a = [sv.window_attention(q, k, v) for _ in range(5)]
    b = [sv.prefix_attention(q, pk, pv, k, v) for _ in range(5)]
    assert all(torch.equal(x, a[0]) for x in a) and all(torch.equal(x, b[0]) for x in b)


def test_long_cache_offsets(sv):
    """Offsets past 2^31 elements: the last row and head of a 5 GiB cache."""
    R, K, C, D = 2, 5, 1 << 21, 128
    k = torch.empty((R, K, C, D), dtype=torch.float16, device=DEV)
    k[1, 4, -700:] = rand((700, D), 33, torch.float16)
    v = k.flip(0)  # other values in the rows read, without a second random fill
    v[1, 4, -700:] = rand((700, D), 34, torch.float16)
    q = rand((R, 1, K, D), 35, torch.float16)
    got = sv.window_attention(q, k, v, window=700)
    want, tol, _, _ = attention(q[1:, :, 4:], k[1:, 4:, -700:].clone(), v[1:, 4:, -700:].clone())
    check(got[1:, :, 4:], want, tol)
    got = sv.window_attention(rand((R, 40, K, D), 36, torch.float16), k, v, window=600)
    want, tol, _, _ = attention(rand((R, 40, K, D), 36, torch.float16)[1:, :, 4:], k[1:, 4:, -700:].clone(),
                                v[1:, 4:, -700:].clone(), window=600)
    check(got[1:, :, 4:], want, tol)


def test_streams_and_graphs(sv):
    """On a side stream, and captured: the graph reads lengths at replay."""
    dtype = torch.bfloat16
    q, k, v = rand((2, 1, 36, 128), 37, dtype), rand((2, 4, 2000, 128), 38, dtype), rand((2, 4, 2000, 128), 39, dtype)
    pk, pv = rand((4, 300, 128), 40, dtype), rand((4, 300, 128), 41, dtype)
    lengths = i32([2000, 900])
    w = torch.zeros((2, 4, 2000), device=DEV)
    want = sv.window_attention(q, k, v, lengths)
    want_p = sv.prefix_attention(q, pk, pv, k, v, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sv.window_attention(q, k, v, lengths)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sv.window_attention(q, k, v, lengths, weights=w)
        got_p = sv.prefix_attention(q, pk, pv, k, v, lengths)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got_p, want_p)
    check(got, *attention(q, k, v, lengths)[:2])
    lengths.copy_(i32([77, 2000]))
    w.zero_()
    graph.replay()
    torch.cuda.synchronize()
    out, tol, wts, wtol = attention(q, k, v, lengths)
    check(got, out, tol)
    check(w, wts, wtol + 2.0 ** -23 * wts + 1e-30)
    check(got_p, *attention(q, k, v, lengths, prefix=(pk, pv))[:2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 3, 130])
def test_negative_and_zero_scale(sv, dtype, n):
    q, k, v = rand((2, n, 6, 80), 50, dtype), rand((2, 2, 210, 80), 51, dtype), rand((2, 2, 210, 80), 52, dtype)
    for scale in (-0.2, 0.0, 1e-4):
        check(sv.window_attention(q, k, v, scale=scale, window=100, sinks=3),
              *attention(q, k, v, None, None, 100, 3, scale)[:2], f"scale {scale}")
        check(sv.prefix_attention(q, k[0], v[0], k, v, scale=scale),
              *attention(q, k, v, scale=scale, prefix=(k[0], v[0]))[:2], f"prefix, scale {scale}")


def test_empty_sizes(sv):
    """No rows, no queries, no slots."""
    dtype = torch.bfloat16
    k = rand((2, 2, 9, 64), 53, dtype)
    assert sv.window_attention(k.new_empty((0, 1, 4, 64)), k[:0], k[:0]).shape == (0, 1, 4, 64)
    assert sv.window_attention(k.new_empty((2, 0, 4, 64)), k, k).shape == (2, 0, 4, 64)
    q = rand((2, 3, 4, 64), 54, dtype)
    assert (sv.window_attention(q, k[:, :, :0], k[:, :, :0]) == 0).all()
    pk, pv = rand((2, 77, 64), 55, dtype), rand((2, 77, 64), 56, dtype)
    got = sv.prefix_attention(q, pk, pv, k[:, :, :0], k[:, :, :0])
    check(got, *attention(q, k[:, :, :1], k[:, :, :1], [0, 0], prefix=(pk, pv))[:2])


def test_large_window_and_sinks(sv):
    """Numbers past the cache and past 31 bits mean no limit."""
    dtype = torch.float16
    for n in (1, 60):
        q, k, v = rand((2, n, 4, 64), 57, dtype), rand((2, 1, 300, 64), 58, dtype), rand((2, 1, 300, 64), 59, dtype)
        want = sv.window_attention(q, k, v)
        starts = i32([0, 100])
        for window, sinks in ((2 ** 40, 0), (300, 0), (2 ** 31 - 1, 2 ** 31 - 1), (10, 2 ** 35), (7, 300)):
            assert torch.equal(sv.window_attention(q, k, v, window=window, sinks=sinks), want)
            check(sv.window_attention(q, k, v, starts=starts, window=window, sinks=sinks),
                  *attention(q, k, v, None, starts)[:2], f"{window} {sinks}")


def test_weights_past_the_kept_scores(sv):
    """Scores beyond 256 MiB are not kept: the weights come from a second product."""
    R, H, K, D, C = 8, 64, 4, 64, 140000
    q, k, v = rand((R, 1, H, D), 60, torch.bfloat16), rand((1, 1, C, D), 61, torch.bfloat16), \
        rand((1, 1, C, D), 62, torch.bfloat16)
    lengths = i32([C - 100 * r for r in range(R)])
    w = torch.zeros((R, K, C), device=DEV)
    got = sv.window_attention(q, k.expand(R, K, -1, -1), v.expand(R, K, -1, -1), lengths, weights=w)
    r = 3
    want, tol, wts, wtol = attention(q[r:r + 1, :, :16], k, v, lengths[r:r + 1])
    check(got[r:r + 1, :, :16], want, tol)
    check(w[r:r + 1, :1], wts, wtol + 2.0 ** -22 * wts + 1e-30)


def test_statuses_and_clamped_lengths(sv):
    dtype = torch.float16
    q, k, v = rand((3, 1, 4, 64), 42, dtype), rand((3, 4, 50, 64), 43, dtype), rand((3, 4, 50, 64), 44, dtype)
    for n in (1, 40):
        x = rand((3, n, 4, 64), 45, dtype)
        status = i32([-1, -1, -1])
        got = sv.window_attention(x, k, v, i32([60, -5, 50]), starts=i32([0, 0, 51]), status=status)
        assert status.tolist() == [8, 8, 8]
        check(got, *attention(x, k, v, [50, 0, 50], [0, 0, 50])[:2])
        sv.prefix_attention(x, k[0, :, :7], v[0, :, :7], k, v, i32([50, 51, 0]), status=status)
        assert status.tolist() == [0, 8, 0]
    assert sv._lib.error_string(8).startswith("a row's length")


def test_refusals(sv):
    dtype = torch.float16
    q, k = rand((2, 1, 4, 64), 46, dtype), rand((2, 2, 50, 64), 47, dtype)
    w = torch.zeros((2, 2, 50), device=DEV)
    ok = dict(q=q, keys=k, values=k)

    def call(**kw):
        return sv.window_attention(**{**ok, **kw})

    for kw in (dict(q=q[0, 0]), dict(keys=k[:1], values=k[:1]), dict(keys=k.float(), values=k.float()),
               dict(keys=k[..., :32], values=k[..., :32]), dict(values=k.clone()[:, :, :49]),
               dict(q=rand((2, 1, 3, 64), 1, dtype)), dict(window=-1), dict(sinks=-2), dict(lengths=0),
               dict(lengths=51), dict(lengths=i32([1, 2, 3])), dict(lengths=torch.ones(2, device=DEV)),
               dict(weights=w[:, :, :49]), dict(weights=w.half()), dict(q=q.double(), keys=k.double(), values=k.double()),
               dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            call(**kw)
    wide = rand((2, 2, 50, 136), 1, dtype)
    for kw in (dict(q=q.cpu()), dict(keys=k.cpu(), values=k.cpu()), dict(out=torch.empty_like(q).float()),
               dict(out=torch.empty((2, 1, 4, 32), dtype=dtype, device=DEV)), dict(status=torch.zeros(2, device=DEV)),
               dict(q=rand((2, 1, 4, 136), 1, dtype), keys=wide, values=wide),
               dict(q=q[..., :60], keys=k[..., :60], values=k[..., :60]),
               dict(keys=wide[..., 1:65], values=wide[..., 1:65]),
               dict(keys=k[:, :, :1].expand(-1, -1, 50, -1), values=k[:, :, :1].expand(-1, -1, 50, -1))):
        with pytest.raises(RuntimeError):
            call(**kw)
    for kw in (dict(prefix_keys=k[0, :1], prefix_values=k[0, :1]), dict(prefix_length=51), dict(prefix_length=-1)):
        with pytest.raises(ValueError):
            sv.prefix_attention(**{**dict(q=q, prefix_keys=k[0], prefix_values=k[0], keys=k, values=k), **kw})


@pytest.mark.parametrize("n", [1, 40])
def test_float_keys_at_the_end_of_the_range(sv, n):
    """Keys that rounding to fewer bits would make infinite, under a scale that keeps the scores ordinary."""
    g = torch.Generator(device="cuda").manual_seed(11)
    q = torch.randn((2, n, 4, 128), generator=g, device="cuda") * 2.0 ** -8
    k = torch.randn((2, 2, 200, 128), generator=g, device="cuda").clamp(-1, 1)
    k[:, :, 5::7] = k[:, :, 5::7].sign()
    k = k * torch.finfo(torch.float32).max
    v = torch.randn((2, 2, 200, 128), generator=g, device="cuda")
    out = sv.window_attention(q, k, v, scale=2.0 ** -124)
    x = q.double().reshape(2, n, 2, 2, 128).permute(0, 2, 3, 1, 4)
    s = torch.einsum("rkgnd,rkcd->rkgnc", x, k.double()) * 2.0 ** -124
    at = torch.arange(200 - n, 200, device="cuda")[:, None]
    s = s.masked_fill(torch.arange(200, device="cuda") > at, float("-inf"))
    want = torch.einsum("rkgnc,rkcd->rkgnd", s.softmax(-1), v.double()).permute(0, 3, 1, 2, 4).reshape(2, n, 4, 128)
    # Products of 128 dimensions with |q k| scale below 1 (2^4 in sum), each within 2^-20 of itself: scores
    # within 2^-16, weights and their sum within 2^-15 of themselves together, outputs as much of the largest value.
    assert torch.isfinite(out).all()
    assert (out.double() - want).abs().max() <= v.abs().max() * 2.0 ** -15
