"""The entry points of the cache held in 4 bits without a GPU: every refusal below returns
its code before any CUDA call."""
import numpy as np
import pytest

from _records_ref import decode, encode, record


def call(fn, base, kw):
    return fn(*{**base, **kw}.values())


WRITE = dict(keys=16, values=32, dtype=1, rows=2, kv_heads=2, tokens=3, head_dim=128, s_row=768, s_head=384, s_tok=128,
             ck=4096, cv=65536, capacity=10, c_row=1600, c_head=800, c_slot=80, lengths=None, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(keys=None), -1), (dict(ck=None), -1), (dict(values=None), -1), (dict(cv=None), -1), (dict(cv=4096), -1),
    (dict(dtype=3), -2), (dict(rows=0), -3), (dict(kv_heads=0), -3), (dict(tokens=-1), -3), (dict(head_dim=100), -3),
    (dict(head_dim=136), -3), (dict(capacity=0), -3), (dict(capacity=2 ** 29 + 1), -3), (dict(tokens=2 ** 29 + 1), -3),
    (dict(rows=40000), -3), (dict(c_slot=64), -3), (dict(c_head=784), -3), (dict(c_row=800), -3), (dict(c_slot=0), -3),
    (dict(c_slot=-80), -3), (dict(c_slot=88), -5), (dict(keys=8), -5), (dict(s_tok=100), -5), (dict(s_head=-384), -5),
    (dict(ck=4104), -5), (dict(tokens=0), 0), (dict(cv=4096 + 80), -3), (dict(cv=4096 + 800), -3), (dict(keys=6000), -1),
    (dict(values=66000), -1),
])
def test_kv_quantize_rejects(sv, kw, code):
    assert call(sv._lib.lib().sv_kv_quantize, WRITE, kw) == code


READ = dict(ck=4096, cv=65536, rows=2, kv_heads=2, head_dim=128, capacity=10, c_row=1600, c_head=800, c_slot=80,
            lengths=None, tokens=3, keys=16, values=32, dtype=1, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(ck=None), -1), (dict(keys=None), -1), (dict(values=None), -1), (dict(cv=None), -1), (dict(values=16), -1),
    (dict(dtype=-1), -2), (dict(tokens=-1), -3), (dict(head_dim=0), -3), (dict(c_slot=0), -3), (dict(c_row=8), -5),
    (dict(keys=24), -5), (dict(keys=4112), -1), (dict(values=65536), -1), (dict(keys=64, values=1088), -1),
])
def test_kv_dequantize_rejects(sv, kw, code):
    assert call(sv._lib.lib().sv_kv_dequantize, READ, kw) == code


ATTEND = dict(q=16, dtype=1, rows=2, tokens=1, heads=16, kv_heads=1, head_dim=128, q_row=2048, q_tok=2048, q_head=128,
              ck=16, cv=16, capacity=1000, c_row=80000, c_head=0, c_slot=80, lengths=None, starts=None, window=0, sinks=0,
              scale=0.1, weights=None, w_row=0, w_head=0, out=65536, ws=None, ws_bytes=0, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(ck=None), -1), (dict(cv=None), -1), (dict(out=None), -1), (dict(dtype=3), -2),
    (dict(rows=0), -3), (dict(heads=15, kv_heads=2), -3), (dict(head_dim=136), -3), (dict(capacity=0), -3),
    (dict(window=-1), -3), (dict(c_slot=0), -3), (dict(c_slot=-80), -3), (dict(c_slot=72), -5), (dict(ck=8), -5),
    (dict(scale=float("nan")), -4), (dict(q_head=-128), -5), (dict(weights=16, w_row=-1), -3), (dict(out=32), -1),
    (dict(ws=None), -6), (dict(ws=16, ws_bytes=8), -6), (dict(capacity=2 ** 29 + 1), -3),
])
def test_quantized_attention_rejects(sv, kw, code):
    assert call(sv._lib.lib().sv_quantized_attention, ATTEND, kw) == code


def test_record_bytes(sv):
    lib = sv._lib.lib()
    assert [lib.sv_kv_record_bytes(d) for d in (8, 32, 40, 64, 72, 96, 128)] == [32, 32, 48, 48, 64, 64, 80]
    assert all(lib.sv_kv_record_bytes(d) == record(d) for d in range(8, 129, 8))
    assert [lib.sv_kv_record_bytes(d) for d in (-8, 0, 4, 100, 136)] == [0] * 5
    assert lib.sv_quantized_attention_workspace_bytes(1, 2, 1, 16, 1, 128, 1000, 0, 0, 0) > 0
    assert lib.sv_quantized_attention_workspace_bytes(1, 2, 1, 16, 3, 128, 1000, 0, 0, 0) == 0


@pytest.mark.parametrize("D", range(8, 129, 8))
def test_values_in_64_bits(D):
    """What a record stands for is within half a step of the value (a step and float16's
    rounding of the pair more at a group's ends)."""
    import torch
    g = np.random.default_rng(D)
    x = g.standard_normal((50, D)) * 2 + 1
    r = encode(x)
    assert r.shape == (50, record(D))
    y = decode(torch.from_numpy(r), D).numpy()
    G = 32 if D > 64 else 16
    for d in range(0, D, G):
        part = x[:, d:d + G]
        step = (part.max(1) - part.min(1)) / 15
        room = step * (0.5 + 15 * 2.0 ** -11) + np.abs(part).max(1) * 2.0 ** -10
        assert (np.abs(y[:, d:d + G] - part) <= room[:, None]).all()
