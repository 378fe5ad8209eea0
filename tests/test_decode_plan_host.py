"""What a recorded decode step keeps of the pages that its sequences share, without a device."""
import types

import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.cache import Cache
from bitnet_c_b200.csrc import ops
from bitnet_c_b200.engine.decode import DecodeRunner
from bitnet_c_b200.engine.few_layers import FewLayers
from bitnet_c_b200.engine.model import Model
from bitnet_c_b200.parts.base import KvRequest


class TwoHeads:
    """A model as far as a DecodeRunner asks: 8 query heads on 2 key/value heads of 64."""

    device = torch.device("cpu")
    fails = False
    few_layers = None

    def shared_heads(self):
        return (8, 2, 64), 0

    def decode_blocks_per_sequence(self):
        return 0

    def shared_pages(self, cache, slots, lengths, native_layer=0):
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


def test_unrecorded_steps_keep_their_plan(monkeypatch):
    cache, slots = cache_of(64 * 5 + 3, 4)
    model, made = TwoHeads(), []

    class Asked(TwoHeads):
        pays = True

        def shared_pages(self, cache, slots, lengths, native_layer=0):
            made.append(list(slots))
            plan = super().shared_pages(cache, slots, lengths, native_layer)
            return plan if self.pays else None

    model = Asked()
    step = lambda which=None: Model._plan_of_step(model, cache, None, list(which or slots), new_tokens(cache, which or slots))  # noqa: E731
    grow = lambda n: [(cache.reserve(s, n), cache.advance(s, n)) for s in slots]  # noqa: E731
    first = step()
    assert first.own_pages == 1 and first.table[:len(first.host)].tolist() == first.host and len(made) == 1
    for pages in (2, 3, 4):
        grow(64)
        assert step() is first and first.own_pages == pages and len(made) == 1
    assert step(slots[:2]) is not first and step().own_pages == 4 and len(made) == 3  # other sequences, and these again
    cache.close(slots.pop())
    assert [r[0] for r in step().runs] == [[0, 1, 2]] and len(made) == 4
    slots += cache.fork(slots[1])
    assert [r[0] for r in step().runs] == [[0, 1, 2, 3], [1, 3]] and len(made) == 5
    monkeypatch.setattr(ops, "USE_SHARED_PAGES", False)
    step()
    assert len(made) == 6
    monkeypatch.undo()
    # an answer of no is kept as well, an error is not
    model.pays = False
    cache.close(slots.pop())
    assert step() is None and step() is None and len(made) == 7
    cache.close(slots.pop())
    model.fails = True
    for _ in range(2):
        with pytest.raises(RuntimeError):
            step()
    assert len(made) == 9
    model.fails, model.pays = False, True
    assert step().runs == [([0, 1], 0, 5)]
    grow(1024)
    step()
    assert len(made) == 11 and step() and len(made) == 11  # asked again after a thousand tokens
    cache.close(slots.pop())
    assert step() is None and len(made) == 11  # nothing is shared any more


def test_unrecorded_steps_that_one_native_call_runs_sooner():
    weights = [torch.empty(shape, dtype=torch.bfloat16, device="meta") for shape in ((768, 1024), (1024, 512), (8192, 1024), (1024, 4096))]
    part = types.SimpleNamespace(w_qkv=weights[0], w_o=weights[1], w_gate_up=weights[2], w_down=weights[3])
    matrices = sum(2 * w.numel() for w in weights)

    class Native(FewLayers):
        def takes(self, model, cache, ctx):
            return ([types.SimpleNamespace(mixer=part, ffn=part)], None, None) if ctx == "few" else None

    class Model2(TwoHeads):
        few_layers, told = Native(), []

        def shared_pages(self, cache, slots, lengths, native_layer):
            self.told.append(native_layer)

    cache, slots = cache_of(64 * 5 + 3, 4)
    positions, model = new_tokens(cache, slots), Model2()
    for ctx in ("few", "few", "many"):  # (what was answered once is kept)
        Model._plan_of_step(model, cache, ctx, slots, positions)
    cache.kept_plan = None
    Model._plan_of_step(model, cache, "many", slots, positions)
    assert model.told == [matrices, 0]
    # the rule: what the native call has the device read
    pages = [list(range(400)) + [1000 + i, 2000 + i] for i in range(64)]
    plan = ops.SharedPlan(pages, 32, 8, 128, "cpu", sms=148)
    assert ops.shared_pays(plan)
    for read, pays in ((720e6 - 1e6, False), (720e6 + 1e6, True)):
        plan.lengths = [402 * 64 // 30]  # (so many pages that the matrices are a part of it)
        plan.native_layer = int(read) - plan.lengths[0] * 64 * 8 * 128 * 4
        assert ops.shared_pays(plan) == pays
