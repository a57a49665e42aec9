"""How much memory a call over a cache held in 4 bits asks for (no GPU needed)."""
import pytest

SCORES, VALUES = 256 << 20, 96 << 20


@pytest.mark.parametrize("dtype,most", [(0, 32), (1, 64), (2, 64)])
@pytest.mark.parametrize("rows,kv,group,tokens,capacity", [(64, 4, 9, 1, 32768), (64, 4, 4, 5, 65536), (1, 8, 4, 8, 300000),
                                                           (1, 1, 1, 1, 1 << 26), (300, 8, 1, 1, 1 << 20)])
def test_scores_of_few_query_rows_are_kept_in_parts(sv, dtype, most, rows, kv, group, tokens, capacity):
    """With accumulated weights, up to 256 MB of scores (or one head's), whatever the rows; no plain values."""
    assert group * tokens <= most
    f = sv._lib.lib().sv_quantized_attention_workspace_bytes
    heads = kv * group
    got = f(dtype, rows, tokens, heads, kv, 128, capacity, 0, 0, 1)
    one = 4 * group * tokens * capacity
    assert got <= max(SCORES, one) + (16 << 20)
    assert got >= min(rows * kv * one, max(one, SCORES // 2))
    assert f(dtype, rows, tokens, heads, kv, 128, capacity, 0, 0, 0) <= 16 << 20
