"""Calls of ``attention_decode_shared`` that give the length bound: the results of those that leave it out, bit for bit."""
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops
from test_attention_shared_gpu import Batch, forked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts,each,shared,tails", [(1, 4, 200, [0, 1, 70, 63]), (3, 5, 1000, [1, 2, 129]), (4, 1, 300, [0, 30])])
def test_with_the_length_bound(cuda_device, prompts, each, shared, tails):
    b = Batch(*forked(prompts, each, shared, tails), 32, 8, 64, cuda_device)
    plan, longest = b.plan(), max(b.pos) + 1
    want = b.check(plan).clone()
    call = lambda *last: ops.attention_decode_shared(b.qkv, 2048, 2560, torch.zeros_like(b.out), len(b.pos), 32, 8, 64, b.scale, b.tok_pos, b.slots, b.table,  # noqa: E731
                                                     b.k, b.v, *last)
    for bound in (longest, longest + 1000):
        assert torch.equal(call(bound, plan), want)
    with pytest.raises(ops.KernelError, match="max_len"):
        call((longest - 1) // 64 * 64, plan)


def test_slots_that_the_kernel_in_front_writes(cuda_device):
    # the sampler lets its successor begin at once, and its tokens are the slots: a call that read them early would find those of the turn before
    b = Batch(*forked(2, 4, 64 * 9, [5, 64 * 3, 130, 0]), 8, 2, 64, cuda_device)
    plan, n = b.plan(), len(b.pos)
    want = b.check(plan).clone()
    rows = b.table.shape[0]
    logits, u = torch.empty((n, rows), device=cuda_device), torch.zeros(n, device=cuda_device)
    table = torch.empty_like(b.table)
    slots, positions = b.slots.clone(), b.tok_pos.clone()
    out = torch.empty_like(b.out)

    def run():
        ops.sample_filtered(logits, 1.0, u=u, out=slots)
        ops.attention_decode_shared(b.qkv, 512, 640, out, n, 8, 2, 64, b.scale, positions, slots, table, b.k, b.v, plan)

    def put(order):  # sequence i in slot order[i]
        logits.fill_(-float("inf"))
        logits[torch.arange(n), order] = 1.0
        table.fill_(b.pages[0][0])  # (every entry names a page: another sequence's would be read)
        table[order] = b.table[b.slots.long()]

    orders = [torch.randperm(rows, generator=torch.Generator().manual_seed(s))[:n].to(cuda_device) for s in range(12)]
    put(orders[0])
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for order in orders[1:]:
        put(order)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(slots.long(), order) and torch.equal(out, want)
    ops.check_tc_status(cuda_device)
