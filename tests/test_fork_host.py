"""Forked sequences without a device: what the copies refuse, and who holds which page."""
import random

import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.cache import Cache, CacheError, CacheFull, PagePool
from bitnet_c_b200.csrc import ops
from bitnet_c_b200.parts import KvRequest


def test_moves_are_grouped_by_source():
    groups, to = ops._page_moves([(4, 0, 9), (7, 1, 64), (4, 8, 9), (4, 2, 11)], 9)
    assert groups == [4, 9, 2, 7, 64, 1, 4, 11, 1] and to == [0, 8, 1, 2]
    assert ops._page_moves([], 3) == ([], [])


@pytest.mark.parametrize("moves,what", [
    ([(9, 0, 1)], "outside"), ([(-1, 0, 1)], "outside"), ([(0, 9, 1)], "outside"), ([(0, 1, 0)], "rows"), ([(0, 1, 65)], "rows"),
    ([(0, 1, 3), (2, 1, 3)], "written once"), ([(0, 1, 3), (1, 2, 3)], "not read"), ([(3, 3, 64)], "not read")])
def test_moves_that_are_refused(moves, what):
    with pytest.raises(ops.KernelError, match=what):
        ops._page_moves(moves, 9)


def test_tensors_that_are_refused():
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_pages(torch.zeros(1, 2, 1, 64, 8), None, [(0, 1, 1)])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.StateSlots([torch.zeros(2, 3)])
    with pytest.raises(ops.KernelError, match="slot"):
        ops.copy_slots(ops.StateSlots([]), 0, [1])


# ---- bookkeeping of forked sequences (no device) -------------------------------------------------
def make(requests, max_tokens=640, max_positions=512, max_seqs=6, states=None):
    return Cache(requests, [None] * len(requests), states or [None] * len(requests), max_tokens, max_positions, torch.bfloat16, None,
                 max_seqs=max_seqs, allocate=False)


def put(c, slot, n):
    c.reserve(slot, n)
    c.advance(slot, n)


@pytest.mark.parametrize("length,shared,own", [(0, 0, 0), (1, 0, 1), (63, 0, 1), (64, 1, 0), (65, 1, 1), (192, 3, 0)])
def test_fork_shares_full_pages_and_takes_one_for_the_rest(length, shared, own):
    c = make([KvRequest(2, 16)])
    g = c.groups[0]
    a = c.open()
    if length:
        put(c, a, length)
    copied = []
    g.copy = copied.extend
    b, d = c.fork(a, 2)
    c.check()
    assert c.length(b) == c.length(d) == length
    assert len(copied) == 2 * own and all(m[2] == length % 64 for m in copied)
    for s in (b, d):
        assert [g.held[s][i] == g.held[a][i] for i in range(shared)] == [True] * shared
        assert len(g.held[s]) == shared + own and (not own or g.held[s][shared] != g.held[a][shared])
    assert g.pool.n_pages - g.pool.n_free == shared + 3 * own
    put(c, b, 70)  # what one writes is nobody else's
    c.check()
    c.close(a)
    c.check()
    c.close(d)
    put(c, b, 1)
    c.check()
    c.close(b)
    assert g.pool.n_free == g.pool.n_pages


def test_fork_without_room_changes_nothing():
    c = make([KvRequest(2, 16), KvRequest(1, 16)], max_tokens=4 * 64, max_seqs=8)
    a = c.open()
    put(c, a, 100)  # two pages of four
    before = [dict(g.held[a]) for g in c.groups], [g.pool.n_free for g in c.groups], c.slots.n_free
    with pytest.raises(CacheFull):
        c.fork(a, 3)
    with pytest.raises(CacheFull):
        c.fork(a, 4)
    c.groups[1].pool.alloc(1)  # the second group has room for one
    with pytest.raises(CacheFull):
        c.fork(a, 2)
    c.groups[1].pool.free([p for p in range(4) if c.groups[1].pool.holders(p) and p not in c.groups[1].held[a].values()])
    assert ([dict(g.held[a]) for g in c.groups], [g.pool.n_free for g in c.groups], c.slots.n_free) == before
    c.check()
    for n in (0, -1):
        with pytest.raises(CacheError, match="at least one"):
            c.fork(a, n)
    with pytest.raises(CacheError, match="not open"):
        c.fork(a + 1)


def test_forks_of_forks_windows_and_compaction_at_random():
    requests = [KvRequest(2, 16), KvRequest(2, 16, window=100), KvRequest(1, 32, window=70, keep_first=5)]
    c = make(requests, max_tokens=64 * 64, max_positions=2000, max_seqs=12)
    rng = random.Random(1)
    live = []
    for turn in range(1500):
        what = rng.random()
        try:
            if what < 0.12 or not live:
                live.append(c.open())
            elif what < 0.3:
                live += c.fork(rng.choice(live), rng.randint(1, 3))
            elif what < 0.45:
                c.close(live.pop(rng.randrange(len(live))))
            elif what < 0.5:
                c.compact()
                for g in c.groups:
                    used = sorted({p for h in g.held.values() for p in h.values()})
                    assert used == list(range(len(used)))
                assert c.compact() == 0
            else:
                put(c, rng.choice(live), rng.choice([1, 1, 30, 64, 130]))
        except CacheFull:
            pass
        c.check()
    for s in live:
        c.close(s)
    assert all(g.pool.n_free == g.pool.n_pages for g in c.groups)


def test_a_pool_counts_its_holders():
    p = PagePool(3)
    a, b = p.alloc(2)
    p.share([a])
    p.free([a])
    assert p.holders(a) == 1 and p.n_free == 1
    p.free([a])
    assert p.holders(a) == 0 and p.n_free == 2
    with pytest.raises(CacheError, match="freed twice"):
        p.free([a])
    with pytest.raises(CacheError, match="shared"):
        p.share([a])
    p.check()


@pytest.mark.parametrize("states", [False, True])
def test_a_copy_that_is_refused_changes_nothing(states):
    """(On the CPU every copy is.)"""
    from bitnet_c_b200.parts import StateRequest
    c = Cache([KvRequest(2, 16)], [None], [StateRequest((3,), torch.float32) if states else None], 640, 512, torch.bfloat16, torch.device("cpu"), max_seqs=6)
    g = c.groups[0]
    a, b = c.open(), c.open()
    put(c, a, 128 if states else 100)
    put(c, b, 10)
    c.close(a)
    a = c.open()
    put(c, a, 130)
    put(c, b, 60)
    c.close(a)
    a = c.open()
    put(c, a, 128 if states else 100)

    def facts():
        return {s: dict(h) for s, h in g.held.items() if h}, g.pool.n_free, c.slots.n_free, c.slots.active(), [c.length(s) for s in c.slots.active()]
    before = facts()
    with pytest.raises(ops.KernelError, match="CUDA"):
        c.fork(a, 2)
    assert facts() == before
    c.check()
    g.pool.alloc(1)
    c.close(a)
    a = c.open()
    put(c, a, 300)
    c.close(b)
    before = facts()
    with pytest.raises(ops.KernelError, match="CUDA"):
        c.compact()
    assert facts() == before
