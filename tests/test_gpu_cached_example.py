"""examples/cached_decoder.py: the cache operators under the drop-in loops.  The logits of
both decodings are compared with the same decoder computed from whole caches in float
(torch operations); the loops then run to their token limit."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(sv):
    spec = importlib.util.spec_from_file_location("cached_decoder", os.path.join(ROOT, "examples", "cached_decoder.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def plain_attention(q, k, v, see):
    """q [R, n, H, D], k / v [R, K, C, D], see [n, C] or [R, n, C]."""
    R, n, H, D = q.shape
    K = k.shape[1]
    s = torch.einsum("rnkgd,rkcd->rkgnc", q.float().unflatten(2, (K, H // K)), k.float()) * D ** -0.5
    s = s.masked_fill(~see.expand(R, n, k.shape[2])[:, None, None], -torch.inf)
    return torch.einsum("rkgnc,rkcd->rnkgd", s.softmax(-1), v.float()).flatten(2, 3).to(q.dtype)


def plain_logits(ex, w, prompt, tokens, window, sinks):
    """Logits after each token, every sequence [prompt, tokens[r]] attended as the decodings
    do: the prompt with a window and sinks, later tokens to everything before."""
    P, R, n = prompt.shape[1], len(tokens), len(tokens[0])
    x = torch.cat([prompt.expand(R, -1, -1), w.embedding[torch.tensor(tokens, device="cuda")]], 1)
    p, j = torch.arange(P + n, device="cuda")[:, None], torch.arange(P + n, device="cuda")
    see = (j <= p) & ((p >= P) | (j > p - window) | (j < sinks))
    out = []
    for m in range(P, P + n + 1):
        out.append(ex.forward(w, x[:, :m], lambda i, q, k, v: plain_attention(q, k, v, see[:m, :m])))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_decodings_match_whole_caches(example, dtype):
    w = example.Weights(dtype=dtype, vocab=256)
    g = torch.Generator(device="cuda").manual_seed(2)
    prompt = torch.randn((1, 130, w.hidden), generator=g, device="cuda").to(dtype)
    tokens = [[5, 9, 200, 31, 7], [11, 3, 3, 90, 64], [5, 1, 0, 255, 12]]
    want = plain_logits(example, w, prompt, tokens, 64, 4)
    # Both sides round the layers' activations to dtype: a few roundings of values of order 1.
    tol = dict(rtol=0, atol=2e-4 if dtype == torch.float32 else 6e-2)
    decoding, first = example.Decoder(w).prefill(prompt, 3, 130 + 5)
    torch.testing.assert_close(first, want[0], **tol)
    parents = torch.arange(3, device="cuda")
    for step in range(5):
        got = decoding.step(torch.tensor([t[step] for t in tokens], device="cuda"))
        torch.testing.assert_close(got, want[step + 1], **tol)
        decoding.reorder_device(parents)
    # Rows 0 and 1 change places, row 2 becomes row 0: the next step continues the parents' rows.
    decoding, _ = example.Decoder(w).prefill(prompt, 3, 130 + 5)
    for step in range(4):
        decoding.step(torch.tensor([t[step] for t in tokens], device="cuda"))
    decoding.reorder_device(torch.tensor([1, 0, 0], device="cuda"))
    got = decoding.step(torch.tensor([tokens[1][4], tokens[0][4], tokens[0][4]], device="cuda"))
    torch.testing.assert_close(got, want[5][[1, 0, 0]], **tol)
    # A budget that is never reached changes nothing.
    decoding, _ = example.Decoder(w, budget=150).prefill(prompt, 1, 200)
    for step in range(5):
        got = decoding.step(torch.tensor([tokens[0][step]], device="cuda"))
        torch.testing.assert_close(got, want[step + 1][:1], **tol)
    weights = decoding.weights[..., :135].sum(-1)
    torch.testing.assert_close(weights, torch.full_like(weights, 5.0 * w.heads / w.kv_heads), rtol=1e-3, atol=1e-3)


def test_loops_run_on_the_example(sv, example):
    from starvector_b200 import runtime_shared as rs
    w = example.Weights()
    g = torch.Generator(device="cuda").manual_seed(3)
    prompt = torch.randn((1, 77, w.hidden), generator=g, device="cuda").to(w.dtype)
    torch.manual_seed(0)
    tokens, why = rs._beam_sample(example.Decoder(w), prompt, 40, 1.0, 0.9, 3, [], None, False, lambda step: None)
    assert len(tokens) == 40 and why == "token_limit"
    tokens, why = rs._sample(example.Decoder(w, budget=90, slack=7), prompt, 60, 1.0, 0.9, [], None, False,
                             lambda step: None)
    assert len(tokens) == 60 and why == "token_limit"


def test_budget_cache_keeps_its_slots(example):
    """After evictions: the budget's slots, the sinks and the recent tokens among them,
    every position once."""
    w = example.Weights()
    g = torch.Generator(device="cuda").manual_seed(4)
    prompt = torch.randn((1, 50, w.hidden), generator=g, device="cuda").to(w.dtype)
    decoding, _ = example.Decoder(w, budget=48, slack=8).prefill(prompt, 1, 400)
    for step in range(40):
        logits = decoding.step(torch.tensor([step], device="cuda"))
    assert torch.isfinite(logits).all() and decoding.length <= 57
    live = decoding.positions[..., :decoding.length]
    assert (decoding.positions[..., decoding.length:] == -1).all()
    for unit in live.reshape(-1, decoding.length).tolist():
        assert len(set(unit)) == decoding.length
        assert set(range(4)) <= set(unit) and set(range(90 - 16, 90)) <= set(unit)
