"""Workspaces and counter slots of paged_attention_q4: one of each for a stream (host logic, no GPU)."""
import gc
import threading
import types

import pytest
import torch

from serving_engine_b200 import q4


@pytest.fixture
def held(monkeypatch):
    """The module's tables, empty, and an allocator that gives host memory."""
    for name in ("_workspaces", "_slots"):
        monkeypatch.setattr(q4, name, {}, raising=False)
    monkeypatch.setattr(q4, "_retired", [])
    empty = torch.empty
    monkeypatch.setattr(q4.torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))


def test_two_threads_first_calls_get_slots_of_their_own(held, monkeypatch):
    """Both are inside the allocation, which releases the interpreter's lock, before either is done."""
    inside = threading.Barrier(2, timeout=20)

    def wait_for_the_other(n, dtype, device):
        inside.wait()
        return torch.zeros(n, dtype=dtype)

    monkeypatch.setattr(q4.torch, "empty", wait_for_the_other)
    got = {}
    threads = [threading.Thread(target=lambda s=s: got.update({s: q4._workspace(0, s, 64)})) for s in (11, 22)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert got[11][1] != got[22][1] and got[11][0].data_ptr() != got[22][0].data_ptr()
    for s in (11, 22):
        assert q4._workspace(0, s, 64) == got[s]  # kept


def test_slots_are_counted_by_device_and_not_handed_out_twice(held):
    slots = [q4._workspace(0, s, 16)[1] for s in range(q4.Q4_COUNTER_SLOTS)]
    assert sorted(slots) == list(range(q4.Q4_COUNTER_SLOTS))
    assert [q4._workspace(1, s, 16)[1] for s in range(3)] == [0, 1, 2]
    with pytest.raises(RuntimeError, match="counter slots of device 0"):
        q4._workspace(0, 10 ** 6, 16)
    assert q4._workspace(0, 5, 16)[1] == slots[5]


def test_a_larger_call_keeps_the_slot_and_the_old_memory(held):
    small = q4._workspace(0, 9, 16)
    large = q4._workspace(0, 9, 64)
    assert large[1] == small[1] and large[0].numel() == 64 and q4._workspace(0, 9, 32)[0] is large[0]
    assert q4._retired[0] is small[0]


def test_workspace_sizes_are_kept_by_device(monkeypatch):
    """Devices may differ in SMs, by which the library sizes the workspace."""
    sizes = iter((100, 900))
    monkeypatch.setattr(q4, "lib", lambda: types.SimpleNamespace(seb_paged_attention_q4_workspace_size=lambda *a: next(sizes)))
    q4._attention_workspace_bytes.cache_clear()
    try:
        assert [q4._attention_workspace_bytes(d, 3, 3, 4, 2, 64) for d in (0, 1, 0)] == [100, 900, 100]
    finally:
        q4._attention_workspace_bytes.cache_clear()


def test_a_workspace_of_its_own(held, monkeypatch):
    """Two graphs captured on one stream, each with its own, hold different memory and counters; the slot
    of one that is gone is handed out again only after the device is idle."""
    synced = []
    monkeypatch.setattr(q4.torch.cuda, "synchronize", synced.append)
    monkeypatch.setattr(q4, "_gone", [])
    monkeypatch.setattr(q4, "_idle", {})
    own = getattr(q4._own, "key", None)
    a, b = q4.Workspace(), q4.Workspace()
    keys = []
    for w in (a, b):
        with w:
            keys.append(q4._own.key)
            with a:
                assert q4._own.key == keys[0]
            assert q4._own.key == keys[-1]
    assert getattr(q4._own, "key", None) == own and keys[0] != keys[1] and max(keys) < 0
    got = [q4._workspace(0, k, 64) for k in (5, *keys)]
    assert len({s for _, s in got}) == 3 and len({w.data_ptr() for w, _ in got}) == 3
    del a
    gc.collect()
    assert q4._gone == [keys[0]]
    rest = [q4._workspace(0, 100 + s, 16)[1] for s in range(q4.Q4_COUNTER_SLOTS - 3)]
    assert not synced and got[1][1] not in rest
    assert q4._workspace(0, 1000, 16)[1] == got[1][1] and synced == [0]
    with pytest.raises(RuntimeError, match="counter slots"):
        q4._workspace(0, 1001, 16)
