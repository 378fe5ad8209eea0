"""Pages and states of a cache copied on the device, against copies made row by row in plain torch."""
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops

pytestmark = pytest.mark.gpu
PAGE = 64


def plain(t, moves):
    out = t.clone()
    for src, dst, rows in moves:
        out[:, dst, :, :rows] = t[:, src, :, :rows]
    return out


def filled(shape, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    if dtype in (torch.uint8, torch.int16):
        return torch.randint(0, 200, shape, generator=g).to(dtype).to(device)
    return torch.randn(shape, generator=g).to(dtype).to(device)


@pytest.mark.parametrize("dtype,k_dim,v_dim,heads", [(torch.bfloat16, 64, 64, 8), (torch.bfloat16, 80, 48, 3), (torch.float32, 192, 64, 1),
                                                     (torch.bfloat16, 5, 7, 2), (torch.float32, 3, 3, 2), (torch.uint8, 33, 0, 1), (torch.int16, 2, 6, 5)])
@pytest.mark.parametrize("rows", [1, 37, 63, 64])
def test_copy_pages(cuda_device, dtype, k_dim, v_dim, heads, rows):
    k = filled((3, 9, heads, PAGE, k_dim), dtype, cuda_device, 1)
    v = filled((3, 9, heads, PAGE, v_dim), dtype, cuda_device, 2) if v_dim else None
    # one source to many, another with other rows, a third alone
    moves = [(4, 0, rows), (4, 8, rows), (7, 1, 64), (4, 2, 11), (3, 6, rows)]
    want = [plain(t, moves) if t is not None else None for t in (k, v)]
    ops.copy_pages(k, v, moves)
    assert torch.equal(k, want[0]) and (v is None or torch.equal(v, want[1]))


@pytest.mark.parametrize("v_heads", [1, 4])
def test_copy_pages_other_value_heads(cuda_device, v_heads):
    k, v = filled((2, 5, 2, PAGE, 16), torch.bfloat16, cuda_device, 1), filled((2, 5, v_heads, PAGE, 48), torch.bfloat16, cuda_device, 2)
    moves = [(0, 3, 20), (1, 4, 64)]
    want = [plain(t, moves) for t in (k, v)]
    ops.copy_pages(k, v, moves)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copy_pages_more_than_one_launch(cuda_device):
    # 700 destinations of one source and 100 single moves: the argument of a launch holds 256
    k = filled((1, 1000, 1, PAGE, 8), torch.bfloat16, cuda_device, 3)
    moves = [(900, d, 9) for d in range(700)] + [(901 + i % 90, 700 + i, 1 + i % 64) for i in range(100)]
    want = plain(k, moves)
    ops.copy_pages(k, None, moves)
    assert torch.equal(k, want)


def test_copy_pages_large_offsets(cuda_device):
    # pages and planes whose offsets pass 32 bits
    k = torch.zeros((5, 4200, 8, PAGE, 128), dtype=torch.float32, device=cuda_device)  # 1.1 GB per plane, 5.5 GB in all
    k[:, 4199] = filled((5, 8, PAGE, 128), torch.float32, cuda_device, 4)
    ops.copy_pages(k, None, [(4199, 4000, 64), (4199, 3, 17)])
    assert torch.equal(k[:, 4000], k[:, 4199]) and torch.equal(k[:, 3, :, :17], k[:, 4199, :, :17]) and not k[:, 3, :, 17:].any()


def test_copy_pages_in_a_graph_on_a_side_stream(cuda_device):
    k = filled((2, 4, 2, PAGE, 64), torch.bfloat16, cuda_device, 5)
    ops.copy_pages(k, None, [(0, 3, 1)])  # compiled and loaded
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        moves = [(0, 1, 30)]
        with torch.cuda.graph(g):
            ops.copy_pages(k, None, moves)
        moves[:] = [(0, 2, 64)]  # the recorded launch has its own copy
        before = k.clone()
        k[:, 0] += 1
        g.replay()
        side.synchronize()
    assert torch.equal(k[:, 1, :, :30], k[:, 0, :, :30]) and torch.equal(k[:, 1, :, 30:], before[:, 1, :, 30:]) and torch.equal(k[:, 2], before[:, 2])


@pytest.mark.parametrize("dtype,shapes", [(torch.float32, [(5, 771), (5, 2, 3), (5, 4096)]), (torch.bfloat16, [(5, 7), (5, 1), (5, 3, 5), (5, 64)]),
                                          (torch.uint8, [(5, 13), (5, 100000)])])
def test_copy_slots(cuda_device, dtype, shapes):
    tensors = [filled(s, dtype, cuda_device, i) for i, s in enumerate(shapes)]
    want = [t.clone() for t in tensors]
    for t in want:
        t[0] = t[4] = t[2]
    ops.copy_slots(ops.StateSlots(tensors), 2, [0, 4])
    assert all(torch.equal(a, b) for a, b in zip(tensors, want))


def test_copy_slots_more_tensors_than_one_launch_takes(cuda_device):
    tensors = [filled((300, 3), torch.float32, cuda_device, i) for i in range(150)]
    want = [t[7].clone() for t in tensors]
    ops.copy_slots(ops.StateSlots(tensors), 7, [i for i in range(300) if i != 7])
    assert all(torch.equal(t, w.expand(300, 3)) for t, w in zip(tensors, want))


# ---- forks of a cache ------------------------------------------------------------------------------
def seen_by(cache, group, slot):
    """Keys and values of the sequence in ``slot``, through the page table on the device: [planes, heads, positions, numbers]."""
    n = cache.length(slot)
    pages = group.page_table[slot, :(n + PAGE - 1) // PAGE].long()
    rows = lambda t: torch.cat([t[:, p] for p in pages], 2)[:, :, :n].clone()
    return rows(group.k), rows(group.v)


@pytest.mark.parametrize("length", [1, 64, 100, 193])
def test_fork_and_compact_keep_what_sequences_see(cuda_device, length):
    from bitnet_c_b200.cache import Cache
    from bitnet_c_b200.parts import KvRequest, StateRequest
    requests = [KvRequest(2, 16), KvRequest(2, 16), KvRequest(1, 32, v_head_dim=48)]
    states = [None, StateRequest((3, 5)), {"a": StateRequest((7,)), "b": StateRequest((2, 4), torch.float32)}]
    c = Cache(requests, [None] * 3, states, 40 * 64, 1000, torch.bfloat16, torch.device(cuda_device), max_seqs=8)
    other = c.open()
    c.reserve(other, 130)
    c.advance(other, 130)
    a = c.open()
    c.reserve(a, length)
    c.advance(a, length)
    for i, g in enumerate(c.groups):
        g.k.copy_(filled(tuple(g.k.shape), g.k.dtype, cuda_device, i))
        g.v.copy_(filled(tuple(g.v.shape), g.v.dtype, cuda_device, i + 9))
    for i, t in enumerate(c.states.values()):
        t.copy_(filled(tuple(t.shape), t.dtype, cuda_device, i))
    c.sync()
    forks = c.fork(a, 3)
    forks += c.fork(forks[1])
    c.sync()
    c.check()
    want = [seen_by(c, g, a) for g in c.groups]
    at_rest = [seen_by(c, g, other) for g in c.groups]

    def same(slots):
        for s in slots:
            for g, w in zip(c.groups, want):
                assert all(torch.equal(x, y) for x, y in zip(seen_by(c, g, s), w))
            assert all(torch.equal(t[s], t[a]) for t in c.states.values())

    same(forks)
    # the last page of each is its own
    if length % PAGE:
        g = c.groups[0]
        g.k[:, int(g.page_table[forks[0], length // PAGE])] = 0
        want_of_first = seen_by(c, g, forks[0])
        assert not torch.equal(want_of_first[0], want[0][0])
        same(forks[1:])
    c.close(forks.pop(0))
    c.close(a)
    left = [seen_by(c, g, forks[0]) for g in c.groups]
    moved = c.compact()
    c.sync()
    c.check()
    assert moved > 0 or length % PAGE == 0
    for g, w, r in zip(c.groups, left, at_rest):
        for s in forks:
            assert all(torch.equal(x, y) for x, y in zip(seen_by(c, g, s), w))
        assert all(torch.equal(x, y) for x, y in zip(seen_by(c, g, other), r))
