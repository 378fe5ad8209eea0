"""Which pages sequences share, and the list of work made of it, without a device."""
import random

import pytest

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops


def test_runs_of_a_tree():
    # all begin with 7; two of them go on with 1 2 3, two others with 4, of which one ends there
    pages = [[7, 1, 2, 3, 9], [7, 1, 2, 3], [7, 4], [7, 4, 5], [8, 1], [], [7]]
    runs, first = ops.shared_runs(pages)
    assert runs == [([0, 1, 2, 3, 6], 0, 1), ([0, 1], 1, 3), ([2, 3], 1, 1)]
    assert first == [4, 4, 2, 2, 0, 0, 1]
    assert ops.shared_runs([]) == ([], []) and ops.shared_runs([[1], [2]]) == ([], [0, 0])
    assert ops.shared_runs([[1, 2], [1, 2], [1, 2]]) == ([([0, 1, 2], 0, 2)], [2, 2, 2])


def pieces_of(plan):
    """For every sequence the pages that its results cover, place by place."""
    h = plan.host
    items, members, sequences = (h[a:] for a in plan.at)
    got = [{} for _ in range(plan.n_seqs)]
    most = ops.SHARED_ROWS // (plan.n_heads // plan.n_kv_heads)
    for i in range(plan.n_items):
        first, count, page, n = items[4 * i:4 * i + 4]
        count, begin = count % 256, count // 256
        if not count:  # what a list of fixed size is padded with
            continue
        assert 1 <= count <= most and n >= 1 and first + count <= plan.n_parts and begin == members[2 * first]
        for m in range(first, first + count):
            b, place = members[2 * m:2 * m + 2]
            assert place not in got[b]
            got[b][place] = list(range(page, page + n))
    return got, [sequences[4 * b:4 * b + 4] for b in range(plan.n_seqs)]  # in the order of their blocks


@pytest.mark.parametrize("heads,kv", [(32, 8), (40, 40), (6, 2), (24, 1), (128, 1), (100, 1)])
@pytest.mark.parametrize("seed", range(6))
def test_every_shared_page_is_read_once_for_every_sequence(heads, kv, seed):
    rng = random.Random(seed)
    pages, ids = [[i] for i in range(rng.randint(1, 3))], 100
    for _ in range(rng.randint(1, 90)):  # forks of forks, each grown a little
        p = list(rng.choice(pages))
        p += range(ids, ids + rng.choice([0, 0, 1, 3, 200]))
        ids += 1000
        pages.append(p)
    pages = [p + [10 ** 6 + i] for i, p in enumerate(pages)]
    plan = ops.SharedPlan(pages, heads, kv, 64, "cpu", sms=148)
    look_over(plan, pages)
    # a list of fixed size for a recorded step
    items, parts = plan.n_items, plan.n_parts
    assert len(plan.pad(items + 5, parts + 9).host) == 4 * (items + 5) + 4 * len(pages) + 2 * (parts + 9)
    look_over(plan, pages)
    with pytest.raises(ops.KernelError, match="do not fit"):
        plan.pad(items, parts)


def look_over(plan, pages):
    got, sequences = pieces_of(plan)
    for first_own, place, n, b in sequences:
        assert sorted(got[b]) == list(range(place, place + n)) and place + n <= plan.n_parts
        assert sorted(x for piece in got[b].values() for x in piece) == list(range(first_own))
        assert first_own < len(pages[b]) and plan.own_pages >= len(pages[b]) - first_own
    order = [s[3] for s in sequences]
    own = [len(p) - f for p, f in zip(pages, plan.first_own)]
    assert sorted(order) == list(range(len(pages))) and [own[b] for b in order] == sorted(own, reverse=True)
    # a run's members really share its pages, and nobody outside begins with them
    for members, first, n in plan.runs:
        begin = pages[members[0]][:first + n]
        assert [b for b in range(len(pages)) if pages[b][:-1][:first + n] == begin] == members


def test_refused():
    for heads, kv, dim in [(6, 4, 64), (8, 0, 64), (129, 1, 64), (8, 8, 40), (8, 8, 144), (8, 8, 0)]:
        with pytest.raises(ops.KernelError, match="not supported"):
            ops.shared_plan([[1], [1]], heads, kv, dim, "cpu")
    with pytest.raises(ops.KernelError, match="without a page"):
        ops.SharedPlan([[1], []], 8, 8, 64, "cpu", sms=148)


@pytest.mark.parametrize("shared,each,prompts,kv,pays", [(64, 4, 1, 8, False), (128, 4, 1, 8, True), (16, 8, 1, 8, False), (32, 8, 1, 8, False), (46, 8, 1, 8, True), (16, 16, 1, 8, True), (4, 64, 1, 8, False),
                                                         (16, 2, 8, 8, False), (32, 2, 8, 8, True), (16, 2, 8, 40, False), (1, 64, 1, 40, False), (0, 64, 1, 8, False)])
def test_where_it_pays(shared, each, prompts, kv, pays):
    pages = [[10 ** 4 * p + i for i in range(shared)] + [10 ** 6 + p * each + e, 10 ** 7 + p * each + e] for p in range(prompts) for e in range(each)]
    assert ops.shared_pays(ops.SharedPlan(pages, 4 * kv, kv, 64, "cpu", sms=148)) == pays
