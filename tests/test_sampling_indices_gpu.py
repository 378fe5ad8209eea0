"""Rows of ``sample_filtered`` whose index names no generator: no token, and no generator is touched for them."""
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops
import plain_sampling

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [7, 5000, 128256])  # one block and clusters
@pytest.mark.parametrize("temperature,top_k", [(0.8, 0), (0.8, 40), (0.0, 0)])
def test_an_index_that_names_no_generator(cuda_device, vocab, temperature, top_k):
    logits = torch.randn(6, vocab, generator=torch.Generator().manual_seed(vocab))
    index = [2, -1, 0, 4, 2 ** 31 - 1, 3]
    states = torch.tensor([1, 2, 3, 4, 99, 98, 97], dtype=torch.int64, device=cuda_device)
    held = states[:4]  # (what lies behind them is another's)
    got = ops.sample_filtered(logits.to(cuda_device), temperature, top_k, rng_state=held, index=torch.tensor(index, dtype=torch.int32, device=cuda_device)).tolist()
    after = [1, 2, 3, 4, 99, 98, 97]
    for r, i in enumerate(index):
        if not 0 <= i < 4:
            assert got[r] == -1
            continue
        after[i], u = plain_sampling.xorshift(after[i])
        want, near = plain_sampling.sample_filtered(logits[r].double().numpy(), temperature, top_k, 1.0, 0.0, u)
        assert near <= 1e-9 or got[r] == want
    assert states.tolist() == after
