"""kv_evict on caches whose keys do not fit a block's shared memory, up to the largest
capacity it accepts: exact, against a restatement in torch operations on the host."""
import pytest
import torch

from test_gpu_evict import run

pytestmark = pytest.mark.gpu
DEV = "cuda"
MOST = 1 << 20


def expected(weights, positions, n, budget, sinks, recent):
    """Slots in their places after the eviction: place[i] is the slot that ends at i."""
    w, p = weights[:n].double(), positions[:n]
    stays = (p < sinks) | (p > int(p.max()) - recent)
    rank = torch.where(stays, torch.inf, torch.where(torch.isnan(w), -torch.inf, w))
    kept = torch.zeros(n, dtype=torch.bool)
    kept[torch.argsort(rank, descending=True, stable=True)[:budget]] = True
    slot = torch.arange(n)
    place = slot[:budget].clone()
    place[~kept[:budget]] = slot[budget:][kept[budget:]]
    return place


@pytest.mark.parametrize("capacity,n,budget,sinks,recent,kind", [
    (MOST, MOST, 1000, 4, 100, "spread"), (MOST, MOST, MOST - 5, 0, 0, "spread"), (MOST, MOST - 1, MOST // 2, 1, 4000, "ties"),
    (MOST, 40, 17, 2, 3, "spread"), (MOST, 500, 1000, 0, 0, "spread"), (600705, 600705, 300001, 4, 64, "ties"),
    (600704, 600704, 2048, 0, 0, "zeros"), (24577, 24577, 24000, 0, 16, "ties"), (999999, 987654, 654321, 5, 7, "nan")])
def test_large_capacities(sv, capacity, n, budget, sinks, recent, kind):
    g = torch.Generator().manual_seed(capacity + n)
    keys = torch.randint(-100, 100, (1, 1, 1, capacity, 8), generator=g).half()
    w = torch.exp(torch.randn(capacity, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, (capacity,), generator=g).float()
    elif kind == "zeros":
        w = torch.zeros(capacity)
    elif kind == "nan":
        w[torch.randint(0, capacity, (capacity // 2,), generator=g)] = torch.nan
    p = torch.randperm(capacity, generator=g).int()
    k, v = keys.to(DEV), (-keys).to(DEV)
    status = torch.full((1,), -1, dtype=torch.int32, device=DEV)
    o = sv.kv_evict(k, v, w.to(DEV).view(1, 1, 1, -1), p.to(DEV).view(1, 1, 1, -1),
                    torch.tensor([n], dtype=torch.int32, device=DEV), budget, sinks=sinks, recent=recent, status=status)
    place = expected(w, p, n, budget, sinks, recent) if n > budget else torch.arange(n)
    m = len(place)
    assert status.item() == 0 and o["lengths"].item() == m
    want = keys.clone()
    want[0, 0, 0, :m] = keys[0, 0, 0, place]
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), -want)
    got_w, got_p = o["weights"].cpu().view(-1), o["positions"].cpu().view(-1)
    assert torch.equal(got_w[:m].view(torch.int32), w[place].view(torch.int32)) and (got_w[m:] == 0).all()
    assert torch.equal(got_p[:m], p[place]) and (got_p[m:] == -1).all()


def test_many_large_units(sv):
    """More than one unit per SM (blocks of 256 threads) and ties past a round of their words."""
    g = torch.Generator(device=DEV).manual_seed(5)
    shape = (1, 1, 300, 25000, 8)
    w = torch.randint(0, 2, shape[:-1], generator=g, device=DEV).float()
    keys = torch.randn(shape, generator=g, device=DEV).half()
    p = torch.argsort(torch.rand(shape[:-1], generator=g, device=DEV), -1).int()
    before = keys.clone()
    o = sv.kv_evict(keys, None, w, p, None, 9000, sinks=4, recent=10)
    for h in (0, 147, 299):
        place = expected(w[0, 0, h].cpu(), p[0, 0, h].cpu(), 25000, 9000, 4, 10).to(DEV)
        assert torch.equal(keys[0, 0, h, :9000], before[0, 0, h][place])
        assert torch.equal(keys[0, 0, h, 9000:], before[0, 0, h, 9000:])
        assert torch.equal(o["positions"][0, 0, h, :9000], p[0, 0, h][place])


def test_restatements_agree(sv):
    """This file's restatement and the slot-by-slot one, where several blocks share a unit."""
    run(sv, (1, 2, 1, 26000, 8), [26000, 25999], 20000, 4, 100,
        weights=torch.randint(0, 5, (1, 2, 1, 26000), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).float())
