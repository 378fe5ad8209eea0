"""Where reading shared pages once pays, for many query heads on few key/value heads (no device): the sides as they were measured."""
import pytest

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops


@pytest.mark.parametrize("heads,kv,dim,pages,each,prompts,pays", [
    # query heads that fit one block of a sequence's own pages: no gain where the results of many places have to be joined
    (16, 1, 128, 32, 64, 1, False), (16, 1, 128, 50, 64, 1, False), (16, 1, 128, 128, 64, 1, True), (16, 1, 128, 256, 16, 1, False),
    (32, 2, 128, 128, 16, 1, False), (32, 2, 128, 256, 16, 1, False), (32, 2, 128, 32, 64, 1, True), (32, 2, 128, 64, 4, 16, True),
    # 24 heads on one: five sequences to a block
    (24, 1, 96, 32, 64, 1, True), (24, 1, 96, 12, 6, 1, False), (24, 1, 96, 128, 4, 1, False), (24, 1, 96, 128, 4, 16, True),
    # more than 64: one sequence to a block, which reads a page once instead of five to eight times
    (71, 1, 64, 32, 64, 1, True), (71, 1, 64, 128, 4, 1, False), (100, 1, 64, 128, 4, 1, False), (100, 1, 64, 32, 64, 1, True), (128, 1, 128, 128, 4, 1, False),
    (128, 1, 128, 256, 4, 1, False), (128, 1, 128, 64, 8, 1, False), (128, 1, 128, 128, 8, 1, True), (128, 1, 128, 128, 64, 1, True), (128, 1, 128, 4, 64, 1, False)])
def test_few_key_value_heads(heads, kv, dim, pages, each, prompts, pays):
    rows = [[10 ** 4 * p + i for i in range(pages)] + [10 ** 6 + p * each + e, 10 ** 7 + p * each + e] for p in range(prompts) for e in range(each)]
    assert ops.shared_pays(ops.SharedPlan(rows, heads, kv, dim, "cpu", sms=148)) == pays
