"""What a recorded decode step keeps of the pages that its sequences share, without a device."""
import types

import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.cache import Cache
from bitnet_c_b200.csrc import ops
from bitnet_c_b200.engine.decode import DecodeRunner
from bitnet_c_b200.parts.base import KvRequest


class TwoHeads:
    """A model as far as a DecodeRunner asks: 8 query heads on 2 key/value heads of 64."""

    device = torch.device("cpu")
    fails = False

    def shared_heads(self):
        return (8, 2, 64), 0

    def decode_blocks_per_sequence(self):
        return 0

    def shared_pages(self, cache, slots, lengths):
        if self.fails:
            raise RuntimeError("no room for the plan")
        return ops.SharedPlan([cache.pages_of(0, s, n // 64 + 1) for s, n in zip(slots, lengths)], 8, 2, 64, "cpu", sms=148)


def cache_of(tokens, n):
    cache = Cache([KvRequest(n_kv_heads=2, head_dim=64)], [None], [None], 64 * 800, 64 * 64, torch.bfloat16, "cpu", max_seqs=12, allocate=False)
    slot = cache.open()
    cache.reserve(slot, tokens)
    cache.advance(slot, tokens)
    return cache, [slot] + cache.fork(slot, n - 1)


def new_tokens(cache, slots):
    for s in slots:
        cache.reserve(s, 1)
    return [cache.length(s) for s in slots]


def test_a_plan_that_could_not_be_made_leaves_no_old_one():
    cache, slots = cache_of(64 * 5 + 3, 4)
    model = TwoHeads()
    runner = DecodeRunner(model, cache, None, 4)
    runner._shared_pages(slots, new_tokens(cache, slots))
    assert runner.ctx.shared.runs == [([0, 1, 2, 3], 0, 5)]
    # one of them ends, and another sequence that shares with nobody takes its slot: the old plan would read the prompt's pages for it
    cache.close(slots[1])
    other = cache.open()
    assert other == slots[1]
    cache.reserve(other, 200)
    cache.advance(other, 200)
    positions = new_tokens(cache, slots)
    model.fails = True
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no room"):
            runner._shared_pages(slots, positions)
        assert runner.ctx.shared is None
    model.fails = False
    runner._shared_pages(slots, positions)
    assert runner.ctx.shared.runs == [([0, 2, 3], 0, 5)] and runner.ctx.shared.first_own == [5, 0, 5, 5]


def test_an_upload_that_failed_is_issued_again(monkeypatch):
    cache, slots = cache_of(64 * 5 + 3, 4)
    runner = DecodeRunner(TwoHeads(), cache, None, 4)
    runner._shared_pages(slots, new_tokens(cache, slots))
    table, first = runner.ctx.shared.table, list(runner.ctx.shared.host)
    cache.close(slots[1])
    cache.open()  # (the same slot)
    cache.reserve(slots[1], 200)
    cache.advance(slots[1], 200)
    positions = new_tokens(cache, slots)
    upload = ops.SharedPlan.upload

    def half(plan, to=None):
        upload(plan, to)
        raise RuntimeError("the copy was cut short")

    monkeypatch.setattr(ops.SharedPlan, "upload", half)
    with pytest.raises(RuntimeError, match="cut short"):
        runner._shared_pages(slots, positions)
    monkeypatch.setattr(ops.SharedPlan, "upload", upload)
    # the first plan again: the buffer of its size holds something else by now
    cache2, slots2 = cache_of(64 * 5 + 3, 4)
    runner.cache = cache2
    assert slots2 == slots
    runner._shared_pages(slots2, new_tokens(cache2, slots2))
    assert runner.ctx.shared.host == first and runner.ctx.shared.table[:len(first)].tolist() == first
    assert runner.ctx.shared.table is table


@pytest.mark.parametrize("n", [2, 12])
def test_recordings_of_growing_sequences(n):
    # what a recording is good for changes with the blocks that share a sequence's own pages, not with every bucket of their number
    cache, slots = cache_of(64 * 5 + 3, n)
    runner = DecodeRunner(TwoHeads(), cache, None, n)
    seen, buckets, splits = set(), set(), set()
    for _ in range(40):
        runner._shared_pages(slots, new_tokens(cache, slots))
        seen.add(runner._shape())
        buckets.add(runner.ctx.shared.own_pages)
        splits.add(runner.ctx.shared.own_splits())
        for s in slots:
            cache.reserve(s, 64)
            cache.advance(s, 64)
    assert len(seen) == len(splits) < len(buckets)
