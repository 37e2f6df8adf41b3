"""StepTables (a step's tables from lengths on the GPU) against a loop over rows, exactly."""
import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from oracle import q4 as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(q_lens, ctx, width, capacity, head, count, pad=0, stride=None, seed=0):
    rng = np.random.default_rng(seed)
    i32 = dict(dtype=torch.int32, device=DEV)
    rows = len(q_lens)
    table = rng.integers(0, 10 ** 6, (rows, stride or width)).astype(np.int32)
    free = rng.permutation(10 * capacity)[:capacity].astype(np.int32)
    total = max(sum(max(q, 0) for q in q_lens) + pad, 1)
    t = b200.StepTables(rows, total, DEV)
    dev_table = torch.tensor(table, device=DEV)
    md = t.build(torch.tensor(q_lens, **i32), torch.tensor(ctx, **i32), dev_table[:, :width], torch.tensor(free, device=DEV),
                 torch.tensor([head, count], **i32))
    want = oracle.step_tables(q_lens, ctx, table[:, :width], free, head, count, total)
    got = (t.q_starts, t.k_lens, t.q_pos_offsets, t.item_row, t.positions, t.slot_mapping, dev_table[:, :width], t.free_state)
    for name, g, w in zip("q_starts k_lens q_pos_offsets item_row positions slot_mapping block_table free_state".split(), got, want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w)), name
    if stride:
        assert np.array_equal(dev_table[:, width:].cpu().numpy(), table[:, width:])
    assert md["total_query"] == total and md["block_table_row_stride"] == width
    return t


@pytest.mark.parametrize("rows", [1, 2, 31, 512, 513, 1500])
@pytest.mark.parametrize("q_max", [1, 5, 60])
def test_steps(rows, q_max):
    rng = np.random.default_rng(rows + q_max)
    q = rng.integers(0, q_max + 1, rows).tolist()
    ctx = rng.integers(0, 200, rows).tolist()
    case(q, ctx, width=17, capacity=rows * 5 + 3, head=int(rng.integers(0, rows * 5 + 3)), count=rows * 5 + 3, pad=3)
    b200.check_device_errors()


def test_boundaries():
    case([1, 1, 1, 16, 17, 0, 0, 15], [0, 15, 16, 0, 0, 16, 0, 17], width=3, capacity=40, head=39, count=20, stride=5)
    case([0, 0], [0, 31], width=2, capacity=1, head=0, count=0)
    b200.check_device_errors()


def test_many_tokens_of_few_rows():
    case([9000, 1, 20000], [7, 100000, 31], width=7000, capacity=2000, head=1990, count=2000)
    b200.check_device_errors()


def test_largest_row_count():
    rows = 16384
    case([1] * rows, list(range(rows)), width=1025, capacity=rows, head=5, count=rows)
    b200.check_device_errors()


def test_free_list_too_short():
    case([20, 20, 1], [0, 3, 16], width=4, capacity=9, head=7, count=3)
    with pytest.raises(RuntimeError, match="too few blocks"):
        b200.check_device_errors()


def test_rows_beyond_the_table():
    case([20, 3], [30, 1], width=3, capacity=9, head=0, count=9)
    with pytest.raises(RuntimeError, match="k_len exceeds"):
        b200.check_device_errors()


def test_bad_lengths_and_state():
    case([-4, 3], [5, -9], width=3, capacity=9, head=0, count=9)
    with pytest.raises(RuntimeError, match="index out of range"):
        b200.check_device_errors()
    i32 = dict(dtype=torch.int32, device=DEV)
    t = b200.StepTables(1, 4, DEV)  # a state outside the ring counts as empty; more tokens than places
    t.build(torch.tensor([6], **i32), torch.tensor([0], **i32), torch.zeros(1, 2, **i32), torch.arange(3, **i32),
            torch.tensor([3, 2], **i32))
    with pytest.raises(RuntimeError):
        b200.check_device_errors()
    assert (t.slot_mapping == -1).all() and t.free_state.tolist() == [0, 0]
    assert t.item_row.tolist() == [0, 0, 0, 0] and t.k_lens.tolist() == [6]
    big = 2 ** 31 - 1
    t.build(torch.tensor([big], **i32), torch.tensor([big], **i32), torch.zeros(1, 2, **i32), torch.arange(3, **i32),
            torch.tensor([0, 3], **i32))
    with pytest.raises(RuntimeError):
        b200.check_device_errors()
    assert t.k_lens.tolist() == [big] and (t.slot_mapping == -1).all()


def test_steps_follow_each_other():
    """Two objects in turn: each step starts from the lengths and the free list that the last one left."""
    i32 = dict(dtype=torch.int32, device=DEV)
    rng = np.random.default_rng(5)
    rows, width, cap = 6, 30, 200
    table = torch.zeros(rows, width, **i32)
    ids = rng.permutation(cap).astype(np.int32)
    free, state, ctx = torch.tensor(ids, device=DEV), torch.tensor([190, cap], **i32), torch.zeros(rows, **i32)
    pair = [b200.StepTables(rows, 60, DEV) for _ in range(2)]
    ref_table, ref_ctx, head, count = np.zeros((rows, width), np.int32), np.zeros(rows, int), 190, cap
    for step in range(12):
        q = rng.integers(0, 11, rows)
        t = pair[step % 2]
        t.build(torch.tensor(q, **i32), ctx, table, free, state)
        want = oracle.step_tables(q, ref_ctx, ref_table, ids, head, count, 60)
        ref_table, (head, count) = want[6], want[7]
        assert np.array_equal(t.slot_mapping.cpu().numpy(), want[5])
        assert t.free_state.tolist() == [head, count]
        ctx, ref_ctx = t.k_lens.clone(), np.asarray(want[1])
        state = t.free_state
    assert np.array_equal(table.cpu().numpy(), ref_table)
    b200.check_device_errors()
    held = ref_table[ref_table > 0]
    assert len(set(held.tolist())) == len(held)


def test_graph_replay():
    i32 = dict(dtype=torch.int32, device=DEV)
    t = b200.StepTables(4, 8, DEV)
    q, ctx, table = torch.ones(4, **i32), torch.tensor([15, 16, 3, 0], **i32), torch.zeros(4, 6, **i32)
    free, state = torch.arange(100, 164, **i32), torch.tensor([0, 64], **i32)
    t.build(q, ctx, table, free, state)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.build(q, ctx, table, free, state)
        state.copy_(t.free_state)
        ctx.copy_(t.k_lens)
    for _ in range(20):
        g.replay()
    assert ctx.tolist() == [35, 36, 23, 20]
    assert state.tolist() == [7, 57]
    b200.check_device_errors()


def test_refusals():
    i32 = dict(dtype=torch.int32, device=DEV)
    for bad in ((0, 4), (4, 0), (16385, 1)):
        with pytest.raises(ValueError, match="rows must be"):
            b200.StepTables(*bad)
    t = b200.StepTables(2, 8, DEV)
    good = dict(q_lens=torch.ones(2, **i32), context_lens=torch.ones(2, **i32), block_table=torch.zeros(2, 4, **i32),
                free_ids=torch.arange(9, **i32), free_state=torch.tensor([0, 9], **i32))
    t.build(**good)
    for change, match in ((dict(q_lens=torch.ones(3, **i32)), "q_lens"), (dict(context_lens=torch.ones(2, device=DEV)), "context_lens"),
                          (dict(block_table=torch.zeros(3, 4, **i32)), "block_table"), (dict(block_table=torch.zeros(2, 0, **i32)), "block_table"),
                          (dict(block_table=torch.zeros(1, 4, **i32).expand(2, 4)), "block_table"),
                          (dict(free_ids=torch.arange(0, **i32)), "free_ids"), (dict(free_state=t.free_state), "own free_state"),
                          (dict(free_state=torch.zeros(2, dtype=torch.int32)), "free_state")):
        with pytest.raises(ValueError, match=match):
            t.build(**{**good, **change})
