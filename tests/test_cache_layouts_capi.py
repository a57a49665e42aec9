"""Layouts that the cache operators' entry points refuse, without a GPU: every refusal
below returns its code before any CUDA call."""
import pytest

from test_cache_capi import EVICT, PREFIX, WINDOW, call


WEIGHED = {**WINDOW, "weights": 16, "w_row": 1000, "out": 1 << 20}


@pytest.mark.parametrize("kw", [
    dict(w_row=0, w_head=0), dict(w_row=0, w_head=1000), dict(kv_heads=2, w_row=1000, w_head=0),
    dict(w_row=999), dict(kv_heads=4, w_row=1000, w_head=1000), dict(kv_heads=4, w_row=1, w_head=2000),
    dict(kv_heads=2, w_row=1999, w_head=1000),
])
def test_accumulated_weights_that_overlap(sv, kw):
    """Rows or heads that would add to the same words."""
    assert call(sv._lib.lib().sv_window_attention, WEIGHED, kw) == -3


@pytest.mark.parametrize("kw", [
    dict(), dict(kv_heads=2, w_row=2000, w_head=1000), dict(kv_heads=2, w_row=1000, w_head=2000),
    dict(rows=1, w_row=0), dict(kv_heads=1, w_row=1003, w_head=0), dict(rows=1, kv_heads=4, w_row=0, w_head=1003),
    dict(rows=1, capacity=1, w_row=0, w_head=0),
])
def test_accumulated_weights_that_lie_apart(sv, kw):
    """Past the layout's check: the next thing that is missing is the workspace."""
    assert call(sv._lib.lib().sv_window_attention, WEIGHED, kw) == -6


@pytest.mark.parametrize("kw", [
    dict(s_layer=0), dict(s_row=0), dict(heads=2, s_head=0), dict(s_slot=0), dict(s_slot=64), dict(s_row=12672),
    dict(s_layer=12800), dict(heads=2, s_head=12800, s_row=12800), dict(layers=1, rows=3, s_layer=0, s_row=6400),
])
def test_evicted_caches_that_overlap(sv, kw):
    """Layers, rows, heads or slots that share memory would be moved by several units at once."""
    assert call(sv._lib.lib().sv_kv_evict, EVICT, kw) == -3


SIZE = 4 * 2 * 2 * 100  # bytes of EVICT's weights, of its positions
APART = {**EVICT, "weights": 1 << 20, "positions": 2 << 20, "lengths": 3 << 20, "w_out": 4 << 20, "p_out": 5 << 20,
         "l_out": 6 << 20, "status": 7 << 20}


@pytest.mark.parametrize("out,into", [(o, i) for o in ("w_out", "p_out", "l_out", "status")
                                      for i in ("weights", "positions", "lengths")])
def test_eviction_outputs_over_inputs(sv, out, into):
    """Every output over every input, from its start, its last word or from a word before it."""
    last = {"weights": SIZE, "positions": SIZE, "lengths": 8}[into] - 4
    size = {"w_out": SIZE, "p_out": SIZE, "l_out": 8, "status": 8}[out]
    for at in (0, last, 4 - size):
        if not (out == "l_out" and into == "lengths" and at == 0):
            assert call(sv._lib.lib().sv_kv_evict, APART, {out: APART[into] + at}) == -1


@pytest.mark.parametrize("a,b", [("w_out", "p_out"), ("l_out", "w_out"), ("status", "p_out"), ("l_out", "status")])
def test_eviction_outputs_over_one_another(sv, a, b):
    assert call(sv._lib.lib().sv_kv_evict, APART, {a: APART[b] + 4}) == -1


@pytest.mark.parametrize("base,kw,code", [
    (WINDOW, dict(), -6), (WINDOW, dict(weights=16, w_row=1000), -1), (WINDOW, dict(q_row=4096), -1),
    (WINDOW, dict(q_row=2048 + 128), -1), (WINDOW, dict(rows=1, q_row=0), -6), (WINDOW, dict(out=32), -1),
    (WINDOW, dict(out=16 + 2 * 2 * 2048 - 16), -1), (WINDOW, dict(out=16 + 2 * 2 * 2048), -6),
    (WINDOW, dict(q=16 + 2 * 2 * 2048 - 16), -1), (WINDOW, dict(q=16 + 2 * 2 * 2048), -6),
    (WINDOW, dict(q=16 + 2 * 2 * 2048, weights=16, w_row=1000), -6), (WINDOW, dict(q_head=0), -1),
    (PREFIX, dict(), -6), (PREFIX, dict(out=32), -1), (PREFIX, dict(q_tok=16, tokens=2), -1),
])
def test_outputs_over_queries(sv, base, kw, code):
    """The same memory throughout, without weights, passes (to the workspace that is missing)."""
    fn = "sv_window_attention" if base is WINDOW else "sv_prefix_attention"
    assert call(getattr(sv._lib.lib(), fn), base, kw) == code
