"""kv_evict against a slot-by-slot restatement: which slots stay, where they move,
ties, NaN, protected positions, lengths below the budget, repeated calls.  Copies and
choices are exact: compared bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(keys, values, weights, positions, lengths, budget, sinks, recent):
    """Per unit, on the host: (keys, values, weights, positions, lengths) after it."""
    k, v = keys.cpu().clone(), values.cpu().clone()
    w_in, p_in = weights.cpu(), positions.cpu()
    w, p = torch.zeros_like(w_in), torch.full_like(p_in, -1)
    Ls, R = k.shape[0], k.shape[1]
    H, C = (k.shape[2], k.shape[3])
    for l in range(Ls):
        for r in range(R):
            n = C if lengths is None else int(lengths[r])
            for h in range(H):
                ww, pp = w_in[l, r, h].tolist(), p_in[l, r, h].tolist()
                order = list(range(n))
                if n > budget:
                    newest = max(pp[:n])

                    def rank(j):
                        if pp[j] < sinks or pp[j] > newest - recent:
                            return float("inf")
                        return float("-inf") if ww[j] != ww[j] else ww[j]

                    stay = set(sorted(range(n), key=lambda j: (-rank(j), j))[:budget])
                    holes = [j for j in range(budget) if j not in stay]
                    order = list(range(budget))
                    for hole, j in zip(holes, sorted(j for j in stay if j >= budget)):
                        order[hole] = j
                idx = torch.tensor(order, dtype=torch.long)
                m = len(order)
                k[l, r, h, :m] = keys[l, r, h].cpu()[idx]
                v[l, r, h, :m] = values[l, r, h].cpu()[idx]
                w[l, r, h, :m] = w_in[l, r, h][idx]
                p[l, r, h, :m] = p_in[l, r, h][idx]
    n = torch.full((R,), C) if lengths is None else lengths.cpu()
    return k, v, w, p, n.clamp(max=budget).int()


def bits(t):
    return t.contiguous().view(torch.uint8)


def run(sv, shape, lengths, budget, sinks, recent, dtype=torch.bfloat16, weights=None, positions=None, seed=0):
    L, R, H, C, D = shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    keys = torch.randn(shape, generator=g, device=DEV).to(dtype)
    values = torch.randn(shape, generator=g, device=DEV).to(dtype)
    if weights is None:
        weights = torch.exp(torch.randn((L, R, H, C), generator=g, device=DEV))
    if positions is None:
        positions = torch.argsort(torch.rand((L, R, H, C), generator=g, device=DEV), -1).int()
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = reference(keys, values, weights, positions, ln, budget, sinks, recent)
    w0, p0 = weights.clone(), positions.clone()
    for _ in range(2):  # a repeated call gives the same again
        o = sv.kv_evict(keys, values, weights, positions, ln, budget, sinks=sinks, recent=recent)
        got = (keys, values, o["weights"], o["positions"], o["lengths"])
        for name, a, b in zip(("keys", "values", "weights", "positions", "lengths"), got, want):
            assert torch.equal(bits(a.cpu()), bits(b)), name
        assert torch.equal(bits(weights), bits(w0)) and torch.equal(positions, p0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shape,lengths,budget,sinks,recent", [
    ((1, 1, 1, 2, 8), None, 1, 0, 0), ((2, 3, 2, 100, 64), [100, 33, 57], 40, 4, 8),
    ((1, 2, 1, 2049, 128), None, 2048, 4, 256), ((3, 2, 1, 1000, 80), [999, 1000], 17, 1, 16),
    ((1, 4, 2, 513, 16), [0, 1, 512, 513], 511, 0, 511), ((1, 1, 3, 5000, 8), [4999], 1024, 0, 0),
    ((2, 1, 1, 33, 128), None, 32, 32, 0), ((1, 2, 1, 64, 128), [40, 64], 64, 2, 2)])
def test_evict_matches_restatement(sv, shape, lengths, budget, sinks, recent, dtype):
    run(sv, shape, lengths, budget, sinks, recent, dtype)


def test_ties_and_special_weights(sv):
    """Equal weights keep the lowest slots; -0 ties with +0; NaN and -inf go first;
    +inf ties with protected slots."""
    shape = (1, 6, 1, 300, 8)
    w = torch.zeros((1, 6, 1, 300), device=DEV)
    w[0, 1] = torch.tensor([0.0, -0.0, 1.0], device=DEV).repeat(100)
    w[0, 2, 0, ::2] = torch.nan
    w[0, 3, 0, 100:250] = torch.inf
    w[0, 4] = -torch.inf
    w[0, 4, 0, 50:60] = torch.nan
    w[0, 5] = torch.arange(300, device=DEV) % 7 - 3.0
    for budget, sinks, recent in ((100, 4, 10), (200, 0, 0), (299, 3, 200)):
        run(sv, shape, None, budget, sinks, recent, weights=w)


def test_repeated_and_extreme_positions(sv):
    """More protected slots than fit (positions repeat), negative and large positions."""
    shape = (1, 3, 1, 200, 8)
    p = torch.zeros((1, 3, 1, 200), dtype=torch.int32, device=DEV)
    p[0, 1] = torch.arange(200, device=DEV) - 100
    p[0, 2] = 2 ** 31 - 1 - torch.arange(200, device=DEV).int()
    for budget, sinks, recent in ((50, 4, 10), (199, 0, 50), (60, 0, 0)):
        run(sv, shape, None, budget, sinks, recent, positions=p)


def test_capacity_beyond_shared_memory(sv):
    run(sv, (1, 1, 2, 40000, 8), [39999], 5000, 4, 100)
    run(sv, (1, 1, 1, 33000, 8), None, 32999, 0, 0)


def test_mqa_views_streams_and_graph(sv):
    """A cache without a head dimension, strided layers, values None, a side stream, a
    captured call whose lengths change."""
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn((4, 2, 500, 64), generator=g, device=DEV).half()
    keys = big[::2, :, 50:450]  # [2, 2, 400, 64], strided
    w = torch.rand((2, 2, 400), generator=g, device=DEV)
    p = torch.arange(400, dtype=torch.int32, device=DEV).expand(2, 2, 400).contiguous()
    before = big.clone()
    lengths = torch.tensor([400, 300], dtype=torch.int32, device=DEV)
    want = reference(keys[:, :, None], keys[:, :, None], w[:, :, None], p[:, :, None], lengths, 128, 4, 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        status = torch.full((2,), -1, dtype=torch.int32, device=DEV)
        o = sv.kv_evict(keys, None, w, p, lengths, 128, sinks=4, recent=32, status=status)
    side.synchronize()
    assert status.tolist() == [0, 0]
    assert torch.equal(keys.cpu(), want[0][:, :, 0]) and torch.equal(o["weights"].cpu(), want[2][:, :, 0])
    assert torch.equal(big[1::2], before[1::2]) and torch.equal(big[:, :, :50], before[:, :, :50])
    big.copy_(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = sv.kv_evict(keys, None, w, p, lengths, 128, sinks=4, recent=32)
    lengths.copy_(torch.tensor([129, 400]))
    graph.replay()
    torch.cuda.synchronize()
    want = reference(before[::2, :, 50:450][:, :, None], before[::2, :, 50:450][:, :, None], w[:, :, None],
                     p[:, :, None], lengths, 128, 4, 32)
    assert torch.equal(keys.cpu(), want[0][:, :, 0]) and torch.equal(o["positions"].cpu(), want[3][:, :, 0])


def test_refusals(sv):
    keys = torch.zeros((1, 2, 1, 20, 8), dtype=torch.float16, device=DEV)
    w = torch.zeros((1, 2, 1, 20), device=DEV)
    p = torch.zeros((1, 2, 1, 20), dtype=torch.int32, device=DEV)
    for kw in (dict(budget=0), dict(budget=21), dict(budget=None), dict(budget=5, sinks=3, recent=3),
               dict(budget=5, sinks=-1), dict(budget=5, recent=-1), dict(budget=5, lengths=21), dict(budget=5, lengths=-1),
               dict(budget=5, weights=w.double()), dict(budget=5, positions=p.long()), dict(budget=5, weights=w[..., :19]),
               dict(budget=5, keys=keys[0]), dict(budget=5, values=keys.float())):
        with pytest.raises(ValueError):
            sv.kv_evict(**{**dict(keys=keys, values=keys, weights=w, positions=p), **kw})
    for kw in (dict(keys=keys.cpu(), values=None), dict(out={"weights": w}), dict(out={"positions": p}),
               dict(keys=keys[..., :4], values=None)):
        with pytest.raises(RuntimeError):
            sv.kv_evict(**{**dict(keys=keys, values=keys, weights=w, positions=p, budget=5), **kw})
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    o = sv.kv_evict(keys, keys.clone(), w, p, torch.tensor([25, -3], device=DEV), 5, status=status)
    assert status.tolist() == [8, 8] and o["lengths"].tolist() == [5, 0]
