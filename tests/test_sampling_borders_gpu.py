"""Rows whose decision lies a little more than 10^-9 of their sum from a border, of two or three numbers that weigh anything: errors of weights do not average out.

A weight is off by 2^-31 of itself at most.  So a running sum is off by 2^-31 of itself, a share of the whole sum by 2^-31 of the whole sum, and what is compared by
less than 2^-30 = 0.93e-9 of it: borders from 1e-9 on are decided as in 64 bits, in which the rows are made (to 10^-15).
"""
import numpy as np
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops

pytestmark = pytest.mark.gpu


def near_rows(n_heavy, seed, n=400_000, span=None, nearest=1e-9, farthest=2.2e-9):
    """Logits of the heavy numbers (``span`` temperatures apart at most), temperatures, the float nearest to the share of all but the last of them, and whether that share
    exceeds it; of rows where those two are ``nearest`` to ``farthest`` apart."""
    rng = np.random.default_rng(seed)
    t = rng.uniform(0.3, 2.0, n).astype(np.float32)
    logits = -np.sort(-rng.uniform(-4.0, 4.0, (n, n_heavy)).astype(np.float32), axis=1)
    if span:
        logits = -np.sort(-(rng.uniform(0.0, span, (n, n_heavy)) * t[:, None]).astype(np.float32), axis=1)
    w = np.exp((logits.astype(np.float64) - logits[:, :1].astype(np.float64)) / t.astype(np.float64)[:, None])
    share = w[:, :-1].sum(1) / w.sum(1)
    u = share.astype(np.float32)
    apart = np.abs(share - u.astype(np.float64))
    # the numbers apart from each other, so that the border is the one between the last two
    some = (apart > nearest) & (apart < farthest) & (np.diff(logits, axis=1) < -0.01).all(1) & (w[:, -1] > 1e-3)
    return logits[some], t[some], u[some], (share > u.astype(np.float64))[some]


@pytest.mark.parametrize("n_heavy,vocab,seed", [(2, 40, 1), (3, 40, 2), (2, 5000, 3), (3, 40003, 4)])
@pytest.mark.parametrize("filters", ["none", "top_k", "top_p"])
def test_borders_between_heavy_numbers(cuda_device, n_heavy, vocab, seed, filters):
    heavy, t, share, exceeds = near_rows(n_heavy, seed)
    rows = min(len(t), 16_000_000 // vocab)
    assert rows >= 350
    rng = np.random.default_rng(seed + 10)
    at = np.stack([rng.permutation(40)[:n_heavy] for _ in range(rows)]) * (vocab // 40)
    logits = torch.full((rows, vocab), -150.0, device=cuda_device)  # (what weighs nothing)
    logits.scatter_(1, torch.from_numpy(at).to(cuda_device), torch.from_numpy(heavy[:rows]).to(cuda_device))
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x[:rows])).to(cuda_device)  # noqa: E731
    if filters == "top_p":  # the last one stays or does not, and is drawn if it does
        got = ops.sample_filtered(logits, put(t), 0, put(share), 0.0, u=torch.full((rows,), 1 - 2.0 ** -20, device=cuda_device))
    else:
        got = ops.sample_filtered(logits, put(t), n_heavy if filters == "top_k" else 0, u=put(share))
    want = np.where(exceeds[:rows], at[:, -2], at[:, -1])
    assert (got.cpu().numpy() == want).all(), int((got.cpu().numpy() != want).sum())


def test_borders_between_two_numbers(cuda_device):
    # Of two numbers the first weighs 1 without an error, so the error of its share is at most a quarter of the other's: 2^-33 = 0.12e-9.  They lie close together, where steps
    # are the finest and what is left of them the largest.
    heavy, t, share, exceeds = near_rows(2, 5, n=6_000_000, span=0.65, nearest=0.2e-9, farthest=1e-9)
    assert len(t) >= 50_000
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda_device)  # noqa: E731
    for top_k in (0, 1):  # (with top-k of a third number that weighs nothing: its path adds weights up key by key)
        logits = torch.cat([put(heavy), torch.full((len(t), 1), -1e9, device=cuda_device)], 1) if top_k else put(heavy)
        got = ops.sample_filtered(logits.contiguous(), put(t), 2 * top_k, u=put(share)).cpu().numpy()
        assert (got == np.where(exceeds, 0, 1)).all(), (top_k, int((got != np.where(exceeds, 0, 1)).sum()), len(t))
