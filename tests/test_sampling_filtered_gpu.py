"""Sampling with temperature, top-k, top-p and min-p against sorted rows in 64 bits.

A token is compared where the plain decision is not within 1e-9 of a border (relative to the row's sum): the kernel's sums are exact to
2^-45 per token and its weights to a few units in the last place of a double, so anything nearer would be decided by rounding.
"""
import numpy as np
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops
import plain_sampling

pytestmark = pytest.mark.gpu


def check(logits, temperature, top_k, top_p, min_p, u, device, **more):
    n = logits.shape[0]
    got = ops.sample_filtered(logits.to(device), *(x.to(device) if isinstance(x, torch.Tensor) else x for x in (temperature, top_k, top_p, min_p)),
                              u=u.to(device), **more).cpu().tolist()
    each = [x.tolist() if isinstance(x, torch.Tensor) else [x] * n for x in (temperature, top_k, top_p, min_p, u)]
    compared = 0
    for r in range(n):
        want, near = plain_sampling.sample_filtered(logits[r].double().numpy(), *(x[r] for x in each))
        if near > 1e-9:
            compared += 1
            assert got[r] == want, (r, [x[r] for x in each], got[r], want, near)
    assert compared >= 0.8 * n  # a row's decision is seldom that near


def rows(n, vocab, spread, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, vocab, generator=g) * spread).to(dtype), torch.rand(n, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 33, 1000, 2049, 4097, 32003, 128256])
@pytest.mark.parametrize("temperature,top_k,top_p,min_p", [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (0.9, 0, 1.0, 0.05),
                                                           (0.8, 100, 0.95, 0.01), (2.0, 1, 0.5, 0.9), (1.0, 5000, 0.999, 0.0), (0.0, 3, 0.5, 0.5)])
def test_parameters_for_all_rows(cuda_device, dtype, vocab, temperature, top_k, top_p, min_p):
    logits, u = rows(5, vocab, 2.0, vocab, dtype)
    check(logits, temperature, top_k, top_p, min_p, u, cuda_device)


@pytest.mark.parametrize("vocab,spread", [(50257, 3.0), (50257, 0.1), (3001, 8.0), (262144, 1.0)])
def test_parameters_per_row(cuda_device, vocab, spread):
    n = 37
    logits, u = rows(n, vocab, spread, 3)
    g = torch.Generator().manual_seed(4)
    r = lambda: torch.rand(n, generator=g)
    temperature = torch.where(r() < 0.1, torch.zeros(n), 0.2 + 2 * r())
    top_k = torch.where(r() < 0.5, (r() * vocab).int(), (r() * 60).int()).int()
    top_p, min_p = torch.where(r() < 0.7, r(), torch.ones(n)), torch.where(r() < 0.5, 0.2 * r(), torch.zeros(n))
    check(logits, temperature, top_k, top_p, min_p, u, cuda_device)
    check(logits, 0.9, top_k, 0.9, min_p, u, cuda_device)  # numbers and tensors together


def test_equal_logits_go_by_index(cuda_device):
    # everything equal; a few levels, each thousands of times; two levels only
    g = torch.Generator().manual_seed(5)
    logits = torch.stack([torch.zeros(40000), torch.randint(0, 4, (40000,), generator=g).float(), torch.randint(0, 2, (40000,), generator=g).float() * 1e-3,
                          torch.full((40000,), -1e30), torch.full((40000,), torch.finfo(torch.float32).min)])
    for case in [(1.0, 0, 1.0, 0.0), (1.0, 17, 1.0, 0.0), (1.0, 39999, 0.5, 0.0), (0.5, 30000, 0.3, 0.3), (0.0, 0, 1.0, 0.0)]:
        for seed in range(3):
            check(logits, *case, torch.rand(5, generator=g), cuda_device)


def test_signed_zeros_are_equal(cuda_device):
    logits = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0], [-0.0, 0.0, -0.0, 0.0, -5.0]])
    for u in (0.0, 0.2, 0.3, 0.5, 0.9):
        check(logits, 1.0, 3, 1.0, 0.0, torch.full((2,), u), cuda_device)
    assert ops.sample_filtered(logits.to(cuda_device), 0.0, u=torch.zeros(2, device=cuda_device)).tolist() == [0, 0]


def test_masked_and_infinite_logits(cuda_device):
    inf, low, nan = float("inf"), torch.finfo(torch.float32).min, float("nan")
    n, V = 9, 5003
    logits, u = rows(n, V, 2.0, 6)
    logits[0, :] = -inf                   # nothing left
    logits[1, :] = nan
    logits[2, :] = -inf
    logits[2, 4999] = -3.0                # one left
    logits[3, :] = low
    logits[3, 7] = 1.0                    # masked by the lowest number
    logits[4, 10:] = -inf
    logits[5, ::2] = nan
    logits[6, [5, 900, 4000]] = inf       # they share everything
    logits[7, :] = low                    # all masked by the lowest number: all alike
    logits[8, :] = -inf
    logits[8, 100:103] = low
    for case in [(1.0, 0, 1.0, 0.0), (0.6, 4, 0.9, 0.02), (0.0, 0, 1.0, 0.0), (1.5, 2, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1e-30, 0, 0.9, 0.0), (1e30, 0, 0.9, 0.0)]:
        check(logits, *case, u, cuda_device)
    got = ops.sample_filtered(logits.to(cuda_device), 1.0, u=u.to(cuda_device)).tolist()
    assert got[0] == got[1] == -1 and got[2] == 4999


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 0.5])
def test_first_and_last_random_numbers(cuda_device, u):
    logits, _ = rows(4, 700, 1.0, 8)
    check(logits, 1.0, 50, 0.9, 0.0, torch.full((4,), u), cuda_device)
    check(logits, 1.0, 0, 1.0, 0.0, torch.full((4,), u), cuda_device)
    assert (ops.sample_filtered(logits.to(cuda_device), 1.0, 1, u=torch.full((4,), u, device=cuda_device)).cpu() == logits.argmax(1)).all()


def test_rows_that_lie_apart_and_a_given_output(cuda_device):
    logits, u = rows(6, 3001, 2.0, 9)
    wide = torch.full((6, 3500), float("nan"), device=cuda_device)
    wide[:, 11:3012] = logits.to(cuda_device)
    out = torch.full((8,), 77, dtype=torch.int32, device=cuda_device)
    got = ops.sample_filtered(wide[:, 11:3012], 0.9, 30, 0.9, u=u.to(cuda_device), out=out)
    assert got is out and out[6:].tolist() == [77, 77]
    assert torch.equal(out[:6], ops.sample_filtered(logits.to(cuda_device), 0.9, 30, 0.9, u=u.to(cuda_device)))
    assert torch.equal(wide[:, 11:3012].cpu(), logits)  # read only


def test_own_generators(cuda_device):
    logits, _ = rows(5, 2000, 2.0, 10)
    index = torch.tensor([4, 0, 6, 2, 3], dtype=torch.int32)
    state = torch.tensor([42 + 7919 * i for i in range(7)], dtype=torch.int64)
    dev = state.to(cuda_device)
    host = state.tolist()
    for step in range(3):
        got = ops.sample_filtered(logits.to(cuda_device), 0.8, 50, 0.95, rng_state=dev, index=index.to(cuda_device)).tolist()
        u = []
        for s in index.tolist():
            host[s], x = plain_sampling.xorshift(host[s])
            u.append(x)
        want = ops.sample_filtered(logits.to(cuda_device), 0.8, 50, 0.95, u=torch.tensor(u, device=cuda_device)).tolist()
        assert got == want and dev.tolist() == host


@pytest.mark.parametrize("vocab", [500009, 600011])
def test_more_numbers_than_blocks_hold_or_add_up(cuda_device, vocab):
    # 8 blocks hold 430,000 float32 numbers, a longer row is read anew in each pass; from 520,000 on borders are found by the bits of the keys
    logits, u = rows(2, vocab, 2.0, 11)
    check(logits, 1.0, 0, 0.9, 0.0, u, cuda_device)
    check(logits, 0.7, 300, 0.9, 0.01, u, cuda_device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_stay_in_memory_between_passes(cuda_device, dtype):
    # one block a row, rows too long to be held; rows that do not begin on 16 bytes
    n, vocab = 310, 40007
    logits, u = rows(n, vocab, 2.0, 14, dtype)
    g = torch.Generator().manual_seed(15)
    top_k = torch.where(torch.rand(n, generator=g) < 0.5, torch.randint(1, 3000, (n,), generator=g), torch.zeros(n, dtype=torch.int64)).int()
    top_p = torch.rand(n, generator=g)
    check(logits, 0.8, top_k, top_p, 0.001, u, cuda_device)


def test_rows_with_most_tokens_masked(cuda_device):
    # a grammar leaves a few of many tokens; the others are -inf, or the lowest number
    n, vocab = 24, 60000
    logits, u = rows(n, vocab, 2.0, 16)
    keep = torch.rand(n, vocab, generator=torch.Generator().manual_seed(17)) < 2e-3
    for mask in (float("-inf"), torch.finfo(torch.float32).min):
        masked = torch.where(keep, logits, torch.full((), mask))
        for case in [(0.8, 0, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (1.2, 500, 1.0, 0.0), (1.0, 0, 0.95, 0.01), (0.9, 59999, 0.9, 0.0)]:
            check(masked, *case, u, cuda_device)


def test_weights_far_apart(cuda_device):
    # logits that span thousands of units: nearly all weights vanish, top-k and min-p reach into what weighs nothing
    logits, u = rows(16, 30000, 400.0, 18)
    for case in [(1.0, 0, 1.0, 0.0), (1.0, 200, 0.9999, 0.0), (0.3, 0, 1.0, 1e-25), (5.0, 3000, 1.0, 1e-9), (30.0, 0, 0.99, 0.0)]:
        check(logits, *case, u, cuda_device)


def test_in_a_graph_and_on_two_streams(cuda_device):
    logits, u = rows(16, 32000, 3.0, 12)
    x, v = logits.to(cuda_device), u.to(cuda_device)
    want = ops.sample_filtered(x, 0.8, 40, 0.9, 0.01, u=v)
    out = torch.zeros(16, dtype=torch.int32, device=cuda_device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.sample_filtered(x, 0.8, 40, 0.9, 0.01, u=v, out=out)
    g.replay()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    both = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                both.append(ops.sample_filtered(x, 0.8, 40, 0.9, 0.01, u=v))
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(torch.equal(b, want) for b in both)


def test_shares_of_many_draws(cuda_device):
    # 4,096 random numbers, evenly spread: each kept token is drawn in proportion to its weight, to one draw
    logits, _ = rows(1, 900, 1.5, 13)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    got = ops.sample_filtered(logits.expand(n, -1).contiguous().to(cuda_device), 0.9, 20, 1.0, 0.0, u=u.to(cuda_device)).cpu().numpy()
    w = np.exp((logits[0].double().numpy() - logits.max().item()) / np.float64(np.float32(0.9)))
    kept = np.argsort(-w, kind="stable")[:20]
    for t in kept:
        assert abs((got == t).sum() - n * w[t] / w[kept].sum()) <= 1.0
    assert set(got.tolist()) <= set(kept.tolist())


def test_more_rows_than_16_bits_count(cuda_device):
    x = torch.randn((70001, 50), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    u = torch.rand(70001, generator=torch.Generator().manual_seed(3)).to(cuda_device)
    assert torch.equal(ops.sample_filtered(x, 0.8, top_k=1, u=u), x.argmax(1).int())
    k = torch.randint(1, 4, (70001,), generator=torch.Generator().manual_seed(4)).int().to(cuda_device)
    got = ops.sample_filtered(x, 1e-6, top_k=k, u=torch.full_like(u, 0.999))  # (the first two logits of a row may be as good as equal)
    assert (x.gather(1, got[:, None].long())[:, 0] >= x.amax(1) - 2e-5).all()


@pytest.mark.parametrize("n,vocab", [(48, 32000), (80, 40000), (300, 32000)])
def test_more_blocks_than_run_at_once_again_and_again(cuda_device, n, vocab):
    # blocks of a second wave begin while others end: what a block sets at its beginning must be there for all of its warps
    logits, u = rows(n, vocab, 3.0, 21)
    x, u = logits.to(cuda_device), u.to(cuda_device)
    want = ops.sample_filtered(x, 0.9, 0, 0.9, u=u)
    best = ops.sample_filtered(x, 0.9, 1, u=u)
    assert torch.equal(best, x.argmax(1).int())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [ops.sample_filtered(x, 0.9, 0, 0.9, u=u) for _ in range(20)]
    for _ in range(30):
        g.replay()
        assert all(torch.equal(t, want) for t in got)
