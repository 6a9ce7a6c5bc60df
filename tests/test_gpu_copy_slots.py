"""Pages of a state pool copied within it (qllm2_amd/decode.py: copy_slots, SlotPool.fork,
reorder, compact, clear; qpam_copy_slots) against assignments one by one: bit for bit."""

import pytest
import torch

from qllm2_amd.decode import SlotPool, copy_slots

pytestmark = pytest.mark.gpu


def _pool(slots, page, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(slots, *page, device="cuda", generator=g),
            torch.randint(0, 5000, (slots,), device="cuda", generator=g, dtype=torch.int32))


def _want(t, src, dst):
    out = t.clone()
    for s, d in zip(src, dst):
        out[d] = 0 if s < 0 else t[s]
    return out


def _lists(src, dst, how):
    if how == "host":
        return src, dst
    if how == "cpu":
        return torch.tensor(src), torch.tensor(dst)
    return (torch.tensor(v, device="cuda", dtype=how) for v in (src, dst))


def _run(state, pos, src, dst, how):
    want, want_pos = _want(state, src, dst), _want(pos, src, dst)
    copy_slots(state, *_lists(src, dst, how), pos=pos)
    assert torch.equal(state, want) and torch.equal(pos, want_pos)


HOW = ["host", "cpu", torch.int32, torch.int64]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("count", [1, 2, 15, 16, 17, 63, 64, 65, 200, 256, 257, 448, 449, 1000, 1024, 1025, 2600])
def test_any_moves_at_once(gpu_lib, count, how):
    """A random map (pages read by several, onto themselves, cleared, in cycles) of slots among slots that stay."""
    g = torch.Generator().manual_seed(count)
    slots = count + 7
    state, pos = _pool(slots, (3, 100), count)
    dst = torch.randperm(slots, generator=g)[:count].tolist()
    src = torch.randint(-1, slots, (count,), generator=g).tolist()
    _run(state, pos, src, dst, how)


@pytest.mark.parametrize("how", ["host", torch.int32])
@pytest.mark.parametrize("count", [2, 16, 64, 300, 1100])
def test_one_cycle(gpu_lib, count, how):
    state, pos = _pool(count, (2, 2, 16, 16, 2), 1)
    _run(state, pos, [*range(1, count), 0], list(range(count)), how)


@pytest.mark.parametrize("page", [(1,), (3,), (4,), (5,), (255,), (256,), (257,), (1021,), (2, 3, 1, 32, 32, 2)])
def test_pages_of_any_size(gpu_lib, page):
    state, pos = _pool(40, page, 2)
    _run(state, pos, [3, 3, 3, -1, 7, 9, 8], [0, 1, 2, 5, 7, 8, 9], "host")
    _run(state, pos, [3, 3, 3, -1, 7, 9, 8], [0, 1, 2, 5, 7, 8, 9], torch.int32)


@pytest.mark.parametrize("how", ["host", torch.int32])
def test_one_layer_of_a_pool_and_odd_strides(gpu_lib, how):
    """Pages apart by more than their length: what is between them stays."""
    state, _ = _pool(30, (4, 2, 1, 16, 16, 2), 3)
    whole, layer = state.clone(), state[:, 2]
    want = _want(layer, [0, 1, 2, -1], [1, 2, 0, 9])
    copy_slots(layer, *_lists([0, 1, 2, -1], [1, 2, 0, 9], how))
    assert torch.equal(state[:, 2], want)
    for i in (0, 1, 3):
        assert torch.equal(state[:, i], whole[:, i])
    flat = torch.randn(20 * 37 + 1, device="cuda")[1:].view(20, 37)[:, 2:31]   # 4-byte aligned, rows 37 apart
    want = _want(flat, [4, 5], [5, 4])
    copy_slots(flat, *_lists([4, 5], [5, 4], how))
    assert torch.equal(flat, want)


def test_one_slot_and_no_moves(gpu_lib):
    state, pos = _pool(1, (40,), 4)
    keep = state.clone()
    copy_slots(state, [], [], pos=pos)
    copy_slots(state, torch.empty(0, device="cuda", dtype=torch.int32), torch.empty(0, device="cuda", dtype=torch.int32))
    copy_slots(state, [0], [0], pos=pos)
    assert torch.equal(state, keep)
    copy_slots(state, [-1], [0], pos=pos)
    assert not state.any() and not pos.any()


def test_device_entries_outside_the_pool_do_nothing(gpu_lib):
    state, pos = _pool(10, (500,), 5)
    want, want_pos = _want(state, [1], [2]), _want(pos, [1], [2])
    big = 2 ** 31 - 1
    src = torch.tensor([1, 10, -2, big, 3, 4, -big], device="cuda", dtype=torch.int32)
    dst = torch.tensor([2, 0, 5, 6, 10, -1, 7], device="cuda", dtype=torch.int32)
    copy_slots(state, src, dst, pos=pos)
    assert torch.equal(state, want) and torch.equal(pos, want_pos)


def test_device_entries_of_64_bits_outside_the_pool(gpu_lib):
    """Ids that 32 bits would wrap into the pool."""
    state, pos = _pool(10, (500,), 5)
    want = _want(state, [1], [2])
    src = torch.tensor([1, 2 ** 32, -2 ** 32 + 4, -2 ** 32 - 1, 3, 4], device="cuda")
    dst = torch.tensor([2, 0, 5, 6, 2 ** 32 + 7, -2 ** 32 + 8], device="cuda")
    copy_slots(state, src, dst, pos=pos)
    assert torch.equal(state, want)


def test_offsets_past_32_bits(gpu_lib):
    state = torch.zeros(700, 1 << 22, device="cuda")   # 11.7 GB: slots from 512 on start past 2^31 elements
    state[690].normal_()
    state[3].normal_()
    a, b = state[690].clone(), state[3].clone()
    copy_slots(state, [690, 3, 690], [3, 690, 699])
    assert torch.equal(state[3], a) and torch.equal(state[690], b) and torch.equal(state[699], a)
    assert not state[691:699].any() and not state[4:690].any()


def test_large_pages(gpu_lib):
    """A page of more than 2^32 bytes."""
    state = torch.zeros(3, (1 << 30) + 100, device="cuda")
    state[0, -50:] = 3.0
    state[0, :50] = 2.0
    copy_slots(state, [0, 1], [1, 0])
    assert not state[0].any() and torch.equal(state[1, -50:], torch.full((50,), 3.0, device="cuda")) and float(state[1, 0]) == 2.0
    assert float(state[1].sum()) == 250.0 and not state[2].any()


def test_long_pages_of_many_moves(gpu_lib):
    """A page of more pieces than a launch has threads for, 1100 moves (two of them real)."""
    state = torch.zeros(4, 40 << 20, device="cuda")   # 160 MB: 2.6 million 64-byte pieces, 1024 threads each
    state[1, -3:] = 5.0
    state[1, 0] = 7.0
    pos = torch.arange(4, device="cuda", dtype=torch.int32)
    src, dst = torch.full((1100,), 99, device="cuda", dtype=torch.int32), torch.full((1100,), 99, device="cuda", dtype=torch.int32)
    src[3], dst[3], src[1090], dst[1090] = 1, 3, 0, 1
    copy_slots(state, src, dst, pos=pos)
    assert not state[:3].any() and float(state[3].sum()) == 22.0 and float(state[3, 0]) == 7.0 and float(state[3, -1]) == 5.0
    assert pos.tolist() == [0, 0, 2, 1]


def test_streams_and_graphs(gpu_lib):
    """The lists of a captured call are read at each replay."""
    state, pos = _pool(50, (3, 1, 16, 16, 2), 6)
    src = torch.arange(20, device="cuda", dtype=torch.int32)
    dst = src.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_slots(state, src, dst, pos=pos)
    g = torch.Generator().manual_seed(7)
    for _ in range(4):
        s, d = torch.randint(-1, 50, (20,), generator=g).tolist(), torch.randperm(50, generator=g)[:20].tolist()
        src.copy_(torch.tensor(s, dtype=torch.int32)), dst.copy_(torch.tensor(d, dtype=torch.int32))
        want, want_pos = _want(state, s, d), _want(pos, s, d)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(state, want) and torch.equal(pos, want_pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = _want(state, [4], [5])
    with torch.cuda.stream(side):
        copy_slots(state, [4], [5])
    side.synchronize()
    assert torch.equal(state, want)


# ---------------------------------------------------------------- the pool's own calls

def _slots(n=12, max_len=64):
    pool = SlotPool(n, 2, 3, 16, 2, max_len=max_len)
    g = torch.Generator(device="cuda").manual_seed(8)
    states = [[torch.randn(2, 3, 16, 16, 2, device="cuda", generator=g) for _ in range(2)] for _ in range(4)]
    ids = [pool.acquire(10 * (i + 1), st) for i, st in enumerate(states)]
    return pool, ids


def test_pool_fork(gpu_lib):
    pool, ids = _slots()
    before = pool.state.clone()
    kids = pool.fork(ids[1], 3)
    assert len(set(kids)) == 3 and not set(kids) & set(ids) and pool.live == set(ids) | set(kids)
    for k in kids:
        assert torch.equal(pool.state[k], before[ids[1]]) and int(pool.pos[k]) == 20 == pool._host_pos[k]
    for i in ids:
        assert torch.equal(pool.state[i], before[i])
    assert pool.fork(ids[0], 0) == []
    with pytest.raises(RuntimeError, match="free slots"):
        pool.fork(ids[0], 6)
    with pytest.raises(ValueError, match="no sequence"):
        pool.fork(11)
    for k in kids:
        pool.release(k)
    assert len(pool.fork(ids[0], 8)) == 8   # every slot can be had again, once


@pytest.mark.parametrize("device", [False, True])
def test_pool_reorder(gpu_lib, device):
    pool, ids = _slots()
    before, pos = pool.state.clone(), pool.pos.clone()
    slots, parents = [ids[0], ids[1], ids[2]], [ids[1], ids[0], ids[3]]
    pool.reorder(*((torch.tensor(v, device="cuda") for v in (slots, parents)) if device else (slots, parents)))
    for s, p in zip(slots, parents):
        assert torch.equal(pool.state[s], before[p]) and int(pool.pos[s]) == int(pos[p])
    assert torch.equal(pool.state[ids[3]], before[ids[3]])
    for s in ids:   # the host's positions, from which the rotary table grows, are not behind
        assert pool._host_pos[s] >= int(pool.pos[s])
        assert device or pool._host_pos[s] == int(pool.pos[s])
    if not device:
        with pytest.raises(ValueError, match="no sequence"):
            pool.reorder([ids[0]], [11])
        with pytest.raises(ValueError, match="twice"):
            pool.reorder([ids[0], ids[0]], [ids[1], ids[2]])


def test_pool_compact(gpu_lib):
    pool, ids = _slots()
    scratch = pool.reserve(2)
    kids = pool.fork(ids[3], 3)
    for s in (ids[0], ids[2], kids[1]):
        pool.release(s)
    live = sorted(pool.live)
    before, pos, host = pool.state.clone(), pool.pos.clone(), list(pool._host_pos)
    moved = pool.compact()
    new = [moved.get(s, s) for s in live]
    assert sorted(new) == list(range(len(live))) and pool.live == set(new)
    for s, d in zip(live, new):
        assert torch.equal(pool.state[d], before[s]) and int(pool.pos[d]) == int(pos[s]) and pool._host_pos[d] == host[s]
    assert pool.compact() == {}
    rest = [pool.acquire() for _ in range(12 - len(scratch) - len(live))]
    assert not set(rest) & set(new) and not set(rest) & set(scratch)
    with pytest.raises(RuntimeError):
        pool.acquire()


def test_pool_clear_and_release_twice(gpu_lib):
    pool, ids = _slots()
    before = pool.state.clone()
    pool.clear([ids[0], ids[2]])
    assert not pool.state[ids[0]].any() and not pool.state[ids[2]].any() and torch.equal(pool.state[ids[1]], before[ids[1]])
    assert pool.pos[ids].tolist() == [0, 20, 0, 40] == [pool._host_pos[i] for i in ids]
    with pytest.raises(ValueError, match="no sequence"):
        pool.clear([11])
    pool.release(ids[0])
    pool.release(ids[0])
    got = [pool.acquire() for _ in range(9)]
    assert len(set(got)) == 9
