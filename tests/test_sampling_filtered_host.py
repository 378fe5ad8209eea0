"""What sampling with filters refuses, and its plain form, without a device."""
import numpy as np
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops
import plain_sampling


def test_logits_off_the_device_are_refused():
    with pytest.raises(ops.KernelError, match="logits"):
        ops.sample_filtered(torch.zeros(2, 5), 1.0, u=torch.zeros(2))


def test_plain_form_by_hand():
    row = np.log([0.1, 0.4, 0.2, 0.3])
    pick = lambda u, **k: plain_sampling.sample_filtered(row, 1.0, k.get("top_k", 0), k.get("top_p", 1.0), k.get("min_p", 0.0), u)[0]
    assert [pick(u) for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91)] == [1, 1, 3, 3, 2, 2, 0]
    assert [pick(u, top_k=2) for u in (0.57, 0.58)] == [1, 3]
    assert [pick(u, top_p=0.65) for u in (0.57, 0.58, 0.99)] == [1, 3, 3]
    assert [pick(u, min_p=0.51) for u in (0.57, 0.58, 0.99)] == [1, 3, 3]
    assert pick(0.99, min_p=1.0) == 1
    assert plain_sampling.sample_filtered([-np.inf, np.nan], 1.0, 0, 1.0, 0.0, 0.5)[0] == -1
    assert plain_sampling.sample_filtered([1.0, 2.0, 2.0], 0.0, 0, 1.0, 0.0, 0.9)[0] == 1
