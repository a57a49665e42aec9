"""The tile kernel's other paths: blocks that take several pieces of work in turn, blocks of
two query tiles (with a second tile without rows), blocks that take their steps in two
halves, pieces without steps.  A B200's 148 SMs decide which calls come there: two tiles
per block once blocks of one would be more than 148, halves from 1536 slots per block of
one tile on.  Values that are not finite lie in slots that some queries see and some do
not, so that every piece has notes to make and to read.  Bounds: see _attention_ref."""
import pytest
import torch

from _attention_ref import attention, check, visible
from test_gpu_attention import i32, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]

# rows, tokens, heads, kv_heads, head_dim, capacity, window, sinks, pattern of lengths, starts
CASES = {
    # 500 pieces of one tile in blocks of two: the second tile never has rows.
    "rowless second tiles": (500, 20, 2, 1, 64, 150, 0, 0, "full", None),
    "rowless second tiles, window": (300, 13, 8, 2, 128, 200, 40, 3, "ragged", None),
    # 100 pieces of 44 rows, then 100 of 256.
    "last tile of a unit alone": (100, 150, 2, 1, 64, 160, 0, 0, "ragged", None),
    # The same with many steps: a block's first piece has no second tile, its next one has.
    "last tile of a unit alone, long": (100, 150, 2, 1, 64, 1500, 0, 0, "full", None),
    "last tile of a unit alone, long, ragged": (120, 130, 2, 1, 128, 1000, 0, 0, "ragged", None),
    "last tile of a unit alone, window": (60, 288, 3, 1, 128, 1479, 448, 1, "ragged", None),
    "last tile of a unit alone, wide group": (18, 322, 16, 1, 40, 745, 0, 0, "ragged", "padded"),
    # Four in five rows are empty: blocks have empty pieces one after the other, before and after others.
    "empty rows": (900, 20, 2, 1, 64, 100, 0, 0, "holes", None),
    "empty rows, two tiles": (600, 130, 2, 1, 64, 140, 30, 2, "holes", None),
    # Prompts padded in front: whole blocks of queries see nothing.
    "padded prompts": (5, 1500, 8, 4, 128, 1500, 0, 0, "full", "padded"),
    "padded prompts, window": (8, 1100, 6, 3, 64, 1200, 300, 5, "ragged", "padded"),
    # Halves: without splits, and with three of them.
    "halves": (25, 20, 8, 4, 128, 1700, 0, 0, "short", None),
    "halves, window": (50, 60, 4, 2, 64, 2400, 1600, 70, "ragged", "padded"),
    "halves in splits": (5, 25, 32, 8, 64, 6000, 0, 0, "short", None),
    "halves in splits, 128": (20, 70, 2, 2, 128, 8000, 0, 0, "ragged", None),
}


def rows_of(case):
    R, n, _, _, _, C, _, _, lengths, starts = case
    g = torch.Generator().manual_seed(R * C)
    if lengths == "full":
        ends = [C] * R
    elif lengths == "ragged":
        ends = torch.randint(max(n, C // 2), C + 1, (R,), generator=g).tolist()
    elif lengths == "holes":  # one row in five has slots; and two runs of empty ones longer than a round of blocks
        ends = [int(torch.randint(1, C + 1, (1,), generator=g)) if r % 5 == 0 and not 148 <= r < 444 else 0 for r in range(R)]
    else:  # few slots in a long cache: no step, one, two, an odd number
        some = [0, 1, 10, 63, 64, 65, 128, 130, 192, 320, C - 1, C]
        ends = [some[(7 * r) % 12] for r in range(R)]
    begin = [0] * R if starts is None else [(e * (r % 5)) // 5 if r % 7 else e for r, e in enumerate(ends)]
    return ends, begin


def check_seen(got, want, tol, seen, what):
    """got where no infinity is seen; where one is, it is the output."""
    assert torch.isposinf(got[seen].float()).all(), f"{what}: an infinity that is seen"
    got = torch.where(seen, 0.0, got.float())
    check(got, torch.where(seen, 0.0, want), tol, what)


def put_infinities(v, n, ends, begins, window, sinks):
    """An infinity in dimension 3 of three slots of each row and head: which queries see one."""
    R, K, C, _ = v.shape
    seen = torch.zeros((R, K, n), dtype=torch.bool, device=DEV)
    for r in range(R):
        e = ends[r]
        see = visible(n, C, e, min(begins[r], e), window, sinks, DEV)
        for h in range(K):
            for slot in {max(e - n // 2 - h, 0), max(e - 1, 0), max(e - n - 3, 0)}:
                v[r, h, slot, 3] = torch.inf
                seen[r, h] |= see[:, slot]
    return seen


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", CASES)
def test_pieces(sv, name, dtype):
    R, n, H, K, D, C, window, sinks = CASES[name][:8]
    ends, begins = rows_of(CASES[name])
    q, k, v = rand((R, n, H, D), 1, dtype), rand((R, K, C, D), 2, dtype), rand((R, K, C, D), 3, dtype)
    lengths, starts = i32(ends), None if not any(begins) else i32(begins)
    want, tol, wts, wtol = attention(q, k, v, lengths, starts, window, sinks)
    for weigh in (False, True):
        w = torch.zeros((R, K, C), device=DEV) if weigh else None
        status = i32([-1] * R)
        got = sv.window_attention(q, k, v, lengths, starts=starts, window=window, sinks=sinks, weights=w, status=status)
        check(got, want, tol, name)
        assert status.tolist() == [0] * R
    check(w, wts, wtol + 2.0 ** -23 * wts + 1e-30, f"{name}: weights")
    seen = put_infinities(v, n, ends, begins, window, sinks)
    got = sv.window_attention(q, k, v, lengths, starts=starts, window=window, sinks=sinks)
    again = sv.window_attention(q, k, v, lengths, starts=starts, window=window, sinks=sinks)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[..., 3] = seen.repeat_interleave(H // K, 1).transpose(1, 2)
    # An infinity that no query sees may lie in a tile that is read: elsewhere nothing changes.
    finite = torch.where(torch.isinf(v), 0.0, v.float()).to(dtype)
    want, tol, _, _ = attention(q, k, finite, lengths, starts, window, sinks)
    check_seen(got, want, tol, hit, f"{name}: infinities")


# rows, tokens, heads, kv_heads, head_dim, prefix, capacity
PREFIX = {
    "two tiles": (100, 12, 16, 1, 64, 300, 40),        # 150 tiles of prefix queries, own pieces with rowless tiles
    "two tiles, more than one piece": (200, 24, 8, 1, 128, 200, 30),
    "last tile alone": (26, 131, 10, 5, 40, 14, 572),  # of every unit of the own part, with many steps
    "last tile of the prefix alone": (15, 203, 100, 5, 72, 1000, 80),
    "halves": (64, 9, 16, 1, 128, 3300, 20),            # two splits of 1650 slots
    "halves, one split": (40, 40, 8, 1, 64, 1601, 50),  # 100 tiles
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", PREFIX)
def test_prefix_pieces(sv, name, dtype):
    R, n, H, K, D, P, C = PREFIX[name]
    q, k, v = rand((R, n, H, D), 4, dtype), rand((R, K, C, D), 5, dtype), rand((R, K, C, D), 6, dtype)
    pk, pv = rand((K, P, D), 7, dtype), rand((K, P, D), 8, dtype)
    ends = [(11 * r) % (C + 1) for r in range(R)]
    lengths, status = i32(ends), i32([-1] * R)
    got = sv.prefix_attention(q, pk, pv, k, v, lengths, status=status)
    assert status.tolist() == [0] * R
    check(got, *attention(q, k, v, lengths, prefix=(pk, pv))[:2], name)
    seen = put_infinities(v, n, ends, [0] * R, 0, 0)
    got = sv.prefix_attention(q, pk, pv, k, v, lengths)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[..., 3] = seen.repeat_interleave(H // K, 1).transpose(1, 2)
    finite = torch.where(torch.isinf(v), 0.0, v.float()).to(dtype)
    check_seen(got, *attention(q, k, finite, lengths, prefix=(pk, pv))[:2], hit, f"{name}: infinities")
