"""How ``attention_decode_shared`` takes the length bound and the plan, without a device."""
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops

PAGES = [[1, 2, 3], [1, 2, 4], [1, 5]]


def call(*last, **named):
    empty = torch.zeros(1)  # refused behind the plan: it lies on no device
    return ops.attention_decode_shared(empty, 0, 0, empty, 3, 8, 2, 64, 0.1, empty, empty, empty, empty, empty, *last, **named)


def test_the_plan_by_place_and_by_name_with_a_bound_and_without():
    plan = ops.SharedPlan(PAGES, 8, 2, 64, "cpu", sms=148)
    for last, named in [((plan,), {}), ((129, plan), {}), ((192, plan), {}), ((10 ** 6, plan), {}), ((None, plan), {}), ((129,), dict(plan=plan)), ((), dict(plan=plan)),
                        ((), dict(max_len=150, plan=plan))]:
        with pytest.raises(ops.KernelError, match="qkv"):  # the first tensor, which follows the plan
            call(*last, **named)


def test_a_bound_below_the_plans_sequences_and_calls_without_a_plan_are_refused():
    plan = ops.SharedPlan(PAGES, 8, 2, 64, "cpu", sms=148)
    for bound in (0, 1, 128):  # three pages hold 129 tokens at least
        with pytest.raises(ops.KernelError, match="max_len"):
            call(bound, plan)
    for last, named in [((), {}), ((129,), {}), ((129, None), {}), ((None, "plan"), {})]:
        with pytest.raises(ops.KernelError, match="plan must be"):
            call(*last, **named)
    with pytest.raises(ops.KernelError, match="two plans"):
        call(plan, plan)
