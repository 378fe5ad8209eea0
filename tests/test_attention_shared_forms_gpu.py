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
