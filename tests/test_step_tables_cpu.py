"""seb_step_tables' checks of its arrays: they run before anything reaches a GPU."""
import pytest

from serving_engine_b200 import _lib
from serving_engine_b200.build import build

ROWS, TOKENS, WIDTH, CAPACITY = 600, 700, 8, 5000
SIZES = {"q_lens": 4 * ROWS, "context_lens": 4 * ROWS, "block_table": 4 * ROWS * WIDTH, "free_ids": 4 * CAPACITY,
         "free_state": 8, "q_starts": 4 * ROWS, "k_lens": 4 * ROWS, "q_pos_offsets": 4 * ROWS, "item_row": 4 * TOKENS,
         "positions": 8 * TOKENS, "slot_mapping": 8 * TOKENS, "free_next": 8}
INPUTS = ("q_lens", "context_lens", "free_ids", "free_state")


def call(at):
    build()
    return _lib.lib().seb_step_tables(
        at["q_lens"], at["context_lens"], ROWS, TOKENS, at["block_table"], WIDTH, WIDTH, at["free_ids"], CAPACITY,
        at["free_state"], at["q_starts"], at["k_lens"], at["q_pos_offsets"], at["item_row"], at["positions"],
        at["slot_mapping"], at["free_next"], None, None)


def apart():
    """Addresses (nothing reads them) of arrays that touch and do not overlap."""
    at, where = {}, 1 << 20
    for name, size in SIZES.items():
        at[name] = where
        where += size
    return at


@pytest.mark.parametrize("out", [n for n in SIZES if n not in INPUTS])
@pytest.mark.parametrize("other", list(SIZES))
def test_outputs_overlap_nothing(out, other):
    """context_lens = the k_lens of the same call, say: other CTAs would still be reading it."""
    if out == other:
        pytest.skip("one array")
    at = apart()
    at[out] = at[other] + SIZES[other] - 4  # its last word
    assert call(at) == _lib.SEB_EINVAL
    assert b"overlaps" in _lib.lib().seb_last_error()
    at[out] = at[other]
    assert call(at) == _lib.SEB_EINVAL
