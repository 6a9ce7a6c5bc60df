"""The slot pool's bookkeeping on the host (CPU): positions after reorders whose lists are on
the device, slot ids of any integer type.  The copies themselves are tested on the GPU; here
they are assignments, and a list "on the device" is one whose values the pool must not see."""

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qllm2_amd import decode
from qllm2_amd.decode import SlotPool, build_rope_cache


def _pool(monkeypatch, slots=6, max_len=16):
    """A pool without its states: positions on the CPU, copies of host lists as assignments."""
    def copies(state, src, dst, pos=None):
        if torch.is_tensor(src):
            return
        old = pos.clone()
        for s, d in zip(src, dst):
            pos[d] = 0 if s < 0 else old[s]

    monkeypatch.setattr(decode, "copy_slots", copies)
    monkeypatch.setattr(decode, "decode_step", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    pool = SlotPool.__new__(SlotPool)
    pool.__dict__.update(n_slots=slots, n_layers=1, n_heads=1, head_dim=16, n_states=1, device=torch.device("cpu"),
                         state=torch.zeros(slots, 1), pos=torch.zeros(slots, dtype=torch.int32), _host_pos=[0] * slots, _exact=True,
                         rope=build_rope_cache(max_len, 16), _free=list(range(slots - 1, -1, -1)), live=set())
    return pool


def _reorder(pool, slots, parents):
    """reorder with device lists: the positions move as on the device, the pool sees none of it."""
    with FakeTensorMode():
        lists = [torch.empty(len(v), device="cuda", dtype=torch.int32) for v in (slots, parents)]
    pool.reorder(*lists)
    old = pool.pos.clone()
    for s, p in zip(slots, parents):
        pool.pos[s] = old[p]


def _step(pool, slots):
    """What a decode step does with the table and the positions; every position has its row."""
    pool.step(0, None, None, None, None, None)
    assert all(int(pool.pos[s]) < pool.rope.shape[0] for s in pool.live)
    pool.advance(slots)


def test_device_reorders_do_not_grow_the_table(monkeypatch):
    """Searches of short sequences, more steps in all than the table has rows, beside one that stays: no position passes
    the table, which stays as it is (captured graphs hold its address)."""
    pool = _pool(monkeypatch)
    rope = pool.rope
    stays = pool.acquire(2)
    for _ in range(20):
        first = pool.acquire(3)
        beams = [first, *pool.fork(first, 2)]
        for _ in range(4):
            _step(pool, beams)
            _reorder(pool, beams, [beams[1], beams[0], beams[0]])
        for s in beams:
            pool.release(s)
    assert pool.rope is rope and int(pool.pos[stays]) == 2


def test_positions_that_reach_the_end_grow_the_table_in_time(monkeypatch):
    pool = _pool(monkeypatch)
    first = pool.acquire(3)
    beams = [first, *pool.fork(first, 2)]
    for _ in range(60):
        _step(pool, beams)
        _reorder(pool, beams, [beams[2], beams[2], beams[1]])
    assert int(pool.pos.max()) == 63 and 64 <= pool.rope.shape[0] <= 128


def test_a_far_sequence_is_not_read_back_at_every_step(monkeypatch):
    """One live sequence near the table's end, others reordered beside it: the positions come from the device now and
    then, not at each step."""
    pool = _pool(monkeypatch, max_len=64)
    pool.acquire(63)
    beams = [pool.acquire(1), pool.acquire(1)]
    reads = []
    whole = torch.Tensor.tolist
    monkeypatch.setattr(torch.Tensor, "tolist", lambda t: (reads.append(t is pool.pos), whole(t))[1])
    for _ in range(50):
        _step(pool, beams)
        _reorder(pool, beams, beams[::-1])
    assert sum(reads) <= 2 and pool.rope.shape[0] <= 130


def test_a_position_from_another_sequence_counts(monkeypatch):
    """A slot that took over the furthest position, and the sequence it came from gone."""
    pool = _pool(monkeypatch)
    far, near = pool.acquire(14), pool.acquire(1)
    _reorder(pool, [near], [far])
    pool.release(far)
    for _ in range(6):
        _step(pool, [near])
    assert int(pool.pos[near]) == 20 and pool.rope.shape[0] > 16


@pytest.mark.parametrize("kind", [int, np.int64, torch.tensor])
def test_slot_ids_of_any_integer_type(monkeypatch, kind):
    pool = _pool(monkeypatch)
    a = pool.acquire(5)
    kids = pool.fork(kind(a), 2)
    assert pool.live == {a, *kids} and [pool._host_pos[k] for k in kids] == [5, 5]
    for s in (a, *kids):
        pool.release(kind(s))
    assert not pool.live and sorted(pool._free) == list(range(6)) and all(type(s) is int for s in pool._free)
    pool.release(kind(a))   # twice: handed out once
    assert sorted(pool._free) == list(range(6))


@pytest.mark.parametrize("ids", [[1.5, 2], torch.tensor([1.0, 2.0]), torch.tensor([[1, 2]]), [[1], [2]], torch.tensor(1),
                                 torch.tensor([True, False])])
def test_lists_that_are_no_ids_are_refused(ids):
    """Not cut to integers: a slot of 1.5 would be slot 1."""
    with FakeTensorMode():
        state = torch.empty(4, 8, device="cuda")
    for src, dst in ((ids, [0, 3]), ([0, 3], ids)):
        with pytest.raises(ValueError, match="must be one list"):
            decode.copy_slots(state, src, dst)


def test_pool_calls_refuse_lists_that_are_no_ids(monkeypatch):
    pool = _pool(monkeypatch)
    a, b = pool.acquire(), pool.acquire()
    for call in (lambda: pool.reorder([a, b], [0.5, 1]), lambda: pool.reorder(torch.tensor([0.0, 1.0]), [a, b]),
                 lambda: pool.clear([0.5])):
        with pytest.raises(ValueError, match="must be one list"):
            call()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_host_tensors_of_any_integer_type(monkeypatch, dtype):
    pool = _pool(monkeypatch)
    a, b = pool.acquire(3), pool.acquire(5)
    pool.reorder(torch.tensor([a, b], dtype=dtype), torch.tensor([b, a], dtype=dtype))
    assert pool._host_pos[a] == 5 and pool._host_pos[b] == 3
    pool.reorder(torch.tensor([]), [])
    pool.clear(torch.tensor([a], dtype=dtype))
    assert pool.pos[[a, b]].tolist() == [0, 3]
