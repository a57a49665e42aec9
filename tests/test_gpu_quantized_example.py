"""The 4-bit cache in examples/cached_decoder.py under the drop-in loops: every attention call of a
few steps against 64 bits over the records it read, the records against the keys they were
made of, and the loop to its token limit."""
import importlib.util
import os

import pytest
import torch

from _attention_ref import check
from _records_ref import attention, decode, encode, same_values

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(sv):
    spec = importlib.util.spec_from_file_location("cached_decoder", os.path.join(ROOT, "examples", "cached_decoder.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps(sv, example, monkeypatch, dtype):
    w = example.Weights(dtype=dtype, vocab=256)
    g = torch.Generator(device="cuda").manual_seed(5)
    prompt = torch.randn((1, 41, w.hidden), generator=g, device="cuda").to(dtype)
    decoding, first = example.Decoder(w, quantized=True).prefill(prompt, 3, 41 + 6)
    assert first.shape == (3, 256) and decoding.length == 41
    written, attended = [], []
    quantize, attend = sv.kv_quantize, sv.quantized_attention

    def spy_quantize(k, v, ck, cv, length):
        quantize(k, v, ck, cv, length)
        written.append((k.clone(), v.clone(), ck[:, :, length - 1:length].clone(), cv[:, :, length - 1:length].clone()))

    def spy_attend(q, ck, cv, length):
        out = attend(q, ck, cv, length)
        attended.append((q.clone(), ck[:, :, :length].clone(), cv[:, :, :length].clone(), out.clone()))
        return out

    monkeypatch.setattr(sv, "kv_quantize", spy_quantize)
    monkeypatch.setattr(sv, "quantized_attention", spy_attend)
    for step in range(5):
        before = decoding.keys.clone()
        parents = torch.tensor([1, 1, step % 3], device="cuda")
        decoding.reorder_device(parents)
        assert torch.equal(decoding.keys[:, :, :, :decoding.length], before[:, parents][:, :, :, :decoding.length])
        logits = decoding.step(torch.tensor([step, 7, 200 - step], device="cuda"))
        assert logits.shape == (3, 256) and torch.isfinite(logits).all()
    assert len(written) == len(attended) == 5 * len(w.layers)
    for k, v, ck, cv in written:
        assert same_values(ck, encode(k.double().cpu().numpy()), w.head_dim)
        assert same_values(cv, encode(v.double().cpu().numpy()), w.head_dim)
    for q, ck, cv, out in attended:
        want, tol, _, _ = attention(q, decode(ck, w.head_dim), decode(cv, w.head_dim))
        check(out, want, tol)


def test_loop_runs(sv, example):
    from starvector_b200 import runtime_shared as rs
    w = example.Weights()
    g = torch.Generator(device="cuda").manual_seed(6)
    prompt = torch.randn((1, 77, w.hidden), generator=g, device="cuda").to(w.dtype)
    torch.manual_seed(0)
    tokens, why = rs._beam_sample(example.Decoder(w, quantized=True), prompt, 40, 1.0, 0.9, 3, [], None, False,
                                  lambda step: None)
    assert len(tokens) == 40 and why == "token_limit"
