"""The cache operators' entry points without a GPU: every refusal below returns its
code before any CUDA call."""
import pytest


def call(fn, base, kw):
    return fn(*{**base, **kw}.values())


WINDOW = dict(q=16, dtype=1, rows=2, tokens=1, heads=16, kv_heads=1, head_dim=128, q_row=2048, q_tok=2048, q_head=128,
              keys=16, values=16, capacity=1000, kv_row=128000, kv_head=0, kv_slot=128, lengths=None, starts=None,
              window=0, sinks=0, scale=0.1, weights=None, w_row=0, w_head=0, out=16, ws=None, ws_bytes=0, status=None,
              stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(keys=None), -1), (dict(values=None), -1), (dict(out=None), -1), (dict(dtype=3), -2),
    (dict(dtype=-1), -2), (dict(rows=0), -3), (dict(tokens=0), -3), (dict(heads=15, kv_heads=2), -3),
    (dict(kv_heads=0), -3), (dict(head_dim=0), -3), (dict(head_dim=136), -3), (dict(head_dim=100), -3),
    (dict(capacity=0), -3), (dict(rows=65536), -3), (dict(rows=60000, tokens=60000), -3), (dict(window=-1), -3),
    (dict(sinks=-1), -3), (dict(scale=float("nan")), -4), (dict(scale=float("inf")), -4), (dict(q=8), -5),
    (dict(kv_slot=100), -5), (dict(q_head=-128), -5), (dict(out=24), -5), (dict(weights=16, w_row=-1), -3),
    (dict(ws=None), -6), (dict(ws=16, ws_bytes=8), -6),
    (dict(kv_slot=0), -3), (dict(capacity=2 ** 29 + 1), -3),
])
def test_window_attention_rejects(sv, kw, code):
    assert call(sv._lib.lib().sv_window_attention, WINDOW, kw) == code


def test_workspace_sizes(sv):
    lib = sv._lib.lib()
    one = lib.sv_window_attention_workspace_bytes(1, 2, 1, 16, 1, 128, 1000, 0, 0, 0)
    assert one > 0
    assert lib.sv_window_attention_workspace_bytes(1, 2, 1, 16, 1, 128, 1000, 0, 0, 1) > one
    assert lib.sv_window_attention_workspace_bytes(1, 2, 1, 16, 3, 128, 1000, 0, 0, 0) == 0  # refused shapes need none
    assert lib.sv_prefix_attention_workspace_bytes(1, 2, 1, 16, 1, 128, 500, 100) > 0
    assert lib.sv_prefix_attention_workspace_bytes(1, 2, 1, 16, 1, 128, -1, 100) == 0


PREFIX = dict(q=16, dtype=1, rows=2, tokens=1, heads=16, kv_heads=1, head_dim=128, q_row=2048, q_tok=2048, q_head=128,
              pk=16, pv=16, prefix=500, p_head=0, p_slot=128, keys=16, values=16, capacity=100, kv_row=12800, kv_head=0,
              kv_slot=128, lengths=None, scale=0.1, out=16, ws=None, ws_bytes=0, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(pk=None), -1), (dict(pv=None), -1), (dict(prefix=-1), -3), (dict(p_slot=4), -5), (dict(pk=8), -5),
    (dict(ws=None), -6), (dict(dtype=9), -2),
])
def test_prefix_attention_rejects(sv, kw, code):
    assert call(sv._lib.lib().sv_prefix_attention, PREFIX, kw) == code


EVICT = dict(keys=16, values=16, elem=2, layers=2, rows=2, heads=1, capacity=100, head_dim=128, s_layer=25600,
             s_row=12800, s_head=0, s_slot=128, weights=16, positions=16, lengths=None, budget=50, sinks=4, recent=8,
             w_out=32, p_out=32, l_out=None, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(keys=None), -1), (dict(weights=None), -1), (dict(positions=None), -1), (dict(w_out=None), -1),
    (dict(p_out=None), -1), (dict(w_out=16), -1), (dict(p_out=16), -1), (dict(elem=8), -2), (dict(layers=0), -3),
    (dict(capacity=0), -3), (dict(layers=70000), -3), (dict(capacity=2 ** 21), -3), (dict(budget=0), -4),
    (dict(budget=101), -4), (dict(sinks=-1), -4), (dict(sinks=30, recent=30), -4), (dict(head_dim=4), -5),
    (dict(s_slot=100), -5), (dict(keys=24), -5),
])
def test_kv_evict_rejects(sv, kw, code):
    assert call(sv._lib.lib().sv_kv_evict, EVICT, kw) == code
