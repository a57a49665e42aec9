"""Views that the cache operators refuse or copy: broadcast and overlapping dimensions.
What is refused is refused on the host, before anything runs."""
import pytest
import torch

from test_gpu_attention import rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n", [1, 40])
def test_broadcast_accumulated_weights_are_refused(sv, n):
    """An accumulator expanded along its slots, rows or heads: torch refuses both for its own additions."""
    R, K, C = 2, 2, 50
    q, k = rand((R, n, 4, 64), 1, torch.float16), rand((R, K, C, 64), 2, torch.float16)
    one = torch.zeros((R, K, 1), device=DEV)
    for w in (one.expand(R, K, C), torch.zeros((1, K, C), device=DEV).expand(R, K, C),
              torch.zeros((R, 1, C), device=DEV).expand(R, K, C), torch.zeros(1, device=DEV).expand(R, K, C)):
        before = w.clone()
        with pytest.raises(ValueError):
            sv.window_attention(q, k, k, weights=w)
        assert torch.equal(w, before)
    with pytest.raises(RuntimeError):  # the second row starts within the first
        sv.window_attention(q, k, k, weights=torch.zeros(300, device=DEV).as_strided((R, K, C), (C, C, 1)))
    # Size-one dimensions have no stride, and a wider accumulator's rows lie apart.
    w = torch.zeros((1, 1, C + 3), device=DEV).expand(1, 1, C + 3)
    sv.window_attention(q[:1], k[:1, :1], k[:1, :1], weights=w)
    assert abs(w[..., :C].sum().item() - 4 * n) < 1e-2 and (w[..., C:] == 0).all()
    w = torch.zeros((K, R, C + 3), device=DEV).transpose(0, 1)
    sv.window_attention(q, k, k, weights=w)
    assert abs(w[..., :C].sum().item() - R * 4 * n) < 1e-2 and (w[..., C:] == 0).all()


@pytest.mark.parametrize("n", [1, 40])
def test_values_broadcast_along_head_dim(sv, n):
    """One stored value for a whole head_dim: queries are copied out, caches refused."""
    dtype = torch.float16
    q, k, v = rand((2, n, 4, 64), 3, dtype), rand((2, 2, 50, 64), 4, dtype), rand((2, 2, 50, 64), 5, dtype)
    for thin in (q[..., :1], q[:1, :1, :1, :1]):
        wide = thin.expand(2, n, 4, 64)
        assert torch.equal(sv.window_attention(wide, k, v), sv.window_attention(wide.contiguous(), k, v))
        assert torch.equal(sv.prefix_attention(wide, k[0], v[0], k, v),
                           sv.prefix_attention(wide.contiguous(), k[0], v[0], k, v))
    flat = k[..., :1].expand(-1, -1, -1, 64)
    with pytest.raises(ValueError):
        sv.window_attention(q, flat, flat)
    with pytest.raises(ValueError):
        sv.prefix_attention(q, flat[0], flat[0], k, v)
    weights, positions = torch.zeros((1, 2, 2, 50), device=DEV), torch.zeros((1, 2, 2, 50), dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        sv.kv_evict(flat[None], None, weights, positions, budget=20)


def test_evicting_from_a_broadcast_cache_is_refused(sv):
    base = rand((2, 2, 2, 50, 64), 6, torch.float16)
    weights = torch.zeros((2, 2, 2, 50), device=DEV)
    positions = torch.zeros((2, 2, 2, 50), dtype=torch.int32, device=DEV)
    for d in range(4):
        keys = base.narrow(d, 0, 1).expand(2, 2, 2, 50, 64)
        before = keys.clone()
        for values in (None, keys):
            with pytest.raises(RuntimeError):
                sv.kv_evict(keys, values, weights, positions, budget=20)
        assert torch.equal(keys, before)
    # Other orders of the dimensions are layouts like any other.
    keys = rand((50, 2, 2, 2, 64), 7, torch.float16)
    view, want = keys.permute(1, 2, 3, 0, 4), keys.clone().permute(1, 2, 3, 0, 4).contiguous()
    weights.copy_(torch.rand(weights.shape, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV))
    a = sv.kv_evict(view, None, weights, positions, budget=20)
    b = sv.kv_evict(want, None, weights, positions, budget=20)
    assert torch.equal(view, want) and torch.equal(a["weights"], b["weights"])


@pytest.mark.parametrize("shape,lengths,budget", [
    ((32, 8, 4, 130, 16), [130, 129, 65, 64, 0, 200, -1, 100], 64),  # many waves of blocks
    ((2, 3, 1, 5000, 64), [5000, 1001, 900], 1000)])                 # several blocks share a unit
def test_lengths_updated_in_place(sv, shape, lengths, budget):
    """out["lengths"] is `lengths`: every layer, head and part still evicts by the old ones."""
    g = torch.Generator(device=DEV).manual_seed(9)
    keys = torch.randn(shape, generator=g, device=DEV).half()
    weights = torch.rand(shape[:-1], generator=g, device=DEV)
    positions = torch.argsort(torch.rand(shape[:-1], generator=g, device=DEV), -1).int()
    old = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want_keys, want_values = keys.clone(), -keys
    want = sv.kv_evict(want_keys, want_values, weights, positions, old, budget, sinks=4, recent=16)
    for _ in range(5):
        k, v, n = keys.clone(), -keys, old.clone()
        status = torch.full_like(n, -1)
        got = sv.kv_evict(k, v, weights, positions, n, budget, sinks=4, recent=16, out={"lengths": n}, status=status)
        assert got["lengths"] is n and torch.equal(n, want["lengths"])
        assert n.tolist() == [min(max(0, min(x, shape[3])), budget) for x in lengths]
        assert status.tolist() == [0 if 0 <= x <= shape[3] else 8 for x in lengths]
        assert torch.equal(k, want_keys) and torch.equal(v, want_values)
        assert torch.equal(got["weights"], want["weights"]) and torch.equal(got["positions"], want["positions"])
    with pytest.raises(RuntimeError):
        sv.kv_evict(k, v, weights, positions, n, budget, status=n)


@pytest.mark.parametrize("n", [1, 40])
def test_statuses_need_a_word_per_row(sv, n):
    """One word broadcast over the rows, or rows apart from one another."""
    q, k = rand((3, n, 4, 64), 10, torch.float16), rand((3, 2, 50, 64), 11, torch.float16)
    weights, positions = torch.zeros((1, 3, 2, 50), device=DEV), torch.zeros((1, 3, 2, 50), dtype=torch.int32, device=DEV)
    words = torch.full((3, 2), -1, dtype=torch.int32, device=DEV)
    for status in (words[:1, 0].expand(3), words[:, 0]):
        for call in (lambda: sv.window_attention(q, k, k, status=status),
                     lambda: sv.prefix_attention(q, k[0], k[0], k, k, status=status),
                     lambda: sv.kv_evict(k[None], None, weights, positions, budget=9, status=status)):
            with pytest.raises(RuntimeError):
                call()
    assert (words == -1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_outputs_in_the_queries_place(sv, n, dtype):
    """out is q: the same result, without weights; with them the queries are needed again."""
    q, k, v = rand((3, n, 8, 64), 12, dtype), rand((3, 2, 900, 64), 13, dtype), rand((3, 2, 900, 64), 14, dtype)
    for call in (lambda x, **kw: sv.window_attention(x, k, v, window=400, sinks=3, **kw),
                 lambda x, **kw: sv.prefix_attention(x, k[0], v[0], k, v, **kw)):
        want, x = call(q), q.clone()
        assert call(x, out=x) is x and torch.equal(x, want)
    w = torch.zeros((3, 2, 900), device=DEV)
    x = q.clone()
    with pytest.raises(RuntimeError):
        sv.window_attention(x, k, v, weights=w, out=x)
    both = rand((2, 3, n, 8, 64), 15, dtype)
    with pytest.raises(RuntimeError):
        sv.window_attention(both.view(6, n, 8, 64)[2:5], k, v, out=both.view(6, n, 8, 64)[3:6])
    assert torch.equal(x, q) and (w == 0).all()


def test_sizes_past_31_bits(sv):
    """Sizes whose low 32 bits alone would be taken for a small cache."""
    q, k = rand((1, 1, 2, 64), 16, torch.float16), rand((1, 1, 1, 64), 17, torch.float16)
    many = 2 ** 32 + 1
    wide = k.expand(1, 1, many, 64)
    for call in (lambda: sv.window_attention(q, wide, wide), lambda: sv.prefix_attention(q, wide[0], wide[0], k, k),
                 lambda: sv.prefix_attention(q, k[0], k[0], wide, wide),
                 lambda: sv.kv_evict(wide[None], None, torch.zeros((), device=DEV).expand(1, 1, 1, many),
                                     torch.zeros((), dtype=torch.int32, device=DEV).expand(1, 1, 1, many), budget=1)):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(sv.prefix_attention(q, wide[0], wide[0], k, k, prefix_length=1),
                       sv.prefix_attention(q, k[0], k[0], k, k))


def test_strides_of_single_entries_mean_nothing(sv):
    """Keys and values of one row and head, cut from caches of different capacities."""
    q, big, small = rand((1, 1, 4, 64), 18, torch.float16), rand((1, 1, 90, 64), 19, torch.float16), \
        rand((1, 1, 70, 64), 20, torch.float16)
    k, v = big[:, :, :60], small[:, :, :60]
    want = sv.window_attention(q, k.contiguous(), v.contiguous())
    assert torch.equal(sv.window_attention(q, k, v), want)
    assert torch.equal(sv.prefix_attention(q, k[0], v[0], k, v),
                       sv.prefix_attention(q, k[0].contiguous(), v[0].contiguous(), k, v.contiguous().clone()))
    weights = torch.rand((1, 1, 1, 60), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    positions = torch.arange(60, dtype=torch.int32, device=DEV).view(1, 1, 1, 60)
    a, b = k.contiguous()[None], v.contiguous()[None]
    sv.kv_evict(a, b, weights, positions, budget=20)
    sv.kv_evict(k[None], v[None], weights, positions, budget=20)
    assert torch.equal(k[None], a) and torch.equal(v[None], b)
    with pytest.raises(ValueError):  # where there are two heads the strides count
        sv.window_attention(q, big.expand(1, 2, -1, -1)[:, :, :60], small.repeat(1, 2, 1, 1)[:, :, :60])
