"""Decode attention over shared pages against plain attention in 64 bits.

The kernel rounds the softmax weights to bfloat16 for the product with the values (the sums of the weights keep float32) and the result once more: at most
2^-8 of sum p |v| / sum p, and 2^-8 of the result.  Scores are float32 sums of exact products; what they and the exponentials add is below 2^-13 of
sum p |v| / sum p at these sizes.
"""
import random

import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops

pytestmark = pytest.mark.gpu
PAGE = 64


class Batch:
    """Sequences that share pages as ``pages`` says (ids per sequence), each with its new token at ``pos``; what no sequence may see is NaN."""

    def __init__(self, pages, pos, heads, kv, dim, device, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.pages, self.pos, self.heads, self.kv, self.dim = pages, pos, heads, kv, dim
        n = len(pages)
        pool = max(p for row in pages for p in row) + 2
        self.k, self.v = (torch.full((pool, kv, PAGE, dim), float("nan"), dtype=torch.bfloat16) for _ in range(2))
        for b, row in enumerate(pages):
            for i, p in enumerate(row):
                seen = min(PAGE, pos[b] - i * PAGE)  # rows in front of the new token
                if seen > 0:
                    for c in (self.k, self.v):
                        if not torch.isfinite(c[p, 0, seen - 1, 0]):
                            c[p, :, :seen] = (torch.randn(kv, seen, dim, generator=g) * spread).to(torch.bfloat16)
        self.k = self.k.to(device)
        self.v = self.v.to(device)
        self.pad = 8
        self.qkv = (torch.randn(n, (heads + 2 * kv) * dim + self.pad, generator=g) * spread).to(torch.bfloat16).to(device)
        order = torch.randperm(n + 3, generator=g)[:n].tolist()  # slots in any order
        table = torch.full((n + 3, max(len(r) for r in pages) + 2), -1, dtype=torch.int32)
        for b, row in enumerate(pages):
            table[order[b], :len(row)] = torch.tensor(row, dtype=torch.int32)
        self.table, self.slots = table.to(device), torch.tensor(order, dtype=torch.int32, device=device)
        self.tok_pos = torch.tensor(pos, dtype=torch.int32, device=device)
        self.out = torch.full((n, heads * dim), 7.0, dtype=torch.bfloat16, device=device)
        self.scale = dim ** -0.5

    def plan(self):
        return ops.shared_plan(self.pages, self.heads, self.kv, self.dim, self.k.device)

    def run(self, plan, out=None):
        H, KV, D = self.heads, self.kv, self.dim
        return ops.attention_decode_shared(self.qkv, H * D, (H + KV) * D, self.out if out is None else out, len(self.pages), H, KV, D, self.scale,
                                           self.tok_pos, self.slots, self.table, self.k, self.v, plan)

    def check(self, plan=None):
        H, KV, D = self.heads, self.kv, self.dim
        k, v = self.k.clone(), self.v.clone()
        got = self.run(plan or self.plan())
        worst = 0.0
        for b, row in enumerate(self.pages):
            p, at = row[self.pos[b] // PAGE], self.pos[b] % PAGE
            k[p, :, at] = self.qkv[b, H * D:(H + KV) * D].reshape(KV, D)
            v[p, :, at] = self.qkv[b, (H + KV) * D:(H + 2 * KV) * D].reshape(KV, D)
        assert torch.equal(k.view(torch.int16), self.k.view(torch.int16)) and torch.equal(v.view(torch.int16), self.v.view(torch.int16))
        for b, row in enumerate(self.pages):
            n = self.pos[b] + 1
            keys, values = (torch.cat([c[p] for p in row], 1)[:, :n].double() for c in (k, v))
            q = self.qkv[b, :H * D].double().reshape(KV, H // KV, D)
            w = torch.softmax(torch.einsum("ghd,gpd->ghp", q, keys) * self.scale, 2)
            want = torch.einsum("ghp,gpd->ghd", w, values).reshape(-1)
            size = torch.einsum("ghp,gpd->ghd", w, values.abs()).reshape(-1)
            off = (got[b].double() - want).abs()
            bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -13) * size
            worst = max(worst, float((off / bound).max()))
        assert worst <= 1.0, worst
        ops.check_tc_status(self.k.device)
        return got


def forked(prompts, each, shared, tails, seed=0):
    """Pages and positions of ``each`` sequences behind each of ``prompts`` prompts of ``shared`` tokens; ids are shuffled."""
    rng = random.Random(seed)
    ids = list(range(prompts * (shared // PAGE) + prompts * each * (max(tails) // PAGE + 3)))
    rng.shuffle(ids)
    pages, pos = [], []
    for _ in range(prompts):
        head = [ids.pop() for _ in range(shared // PAGE)]
        for _ in range(each):
            p = shared + tails[len(pages) % len(tails)]
            pages.append(head + [ids.pop() for _ in range(p // PAGE + 1 - len(head))])
            pos.append(p)
    return pages, pos


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 64), (32, 8, 128), (6, 2, 48), (24, 1, 96), (4, 4, 16), (12, 4, 80), (40, 2, 112), (128, 1, 32), (100, 1, 64)])
@pytest.mark.parametrize("prompts,each,shared,tails", [(1, 2, 64, [0]), (1, 4, 200, [0, 1, 70, 63]), (2, 3, 64 * 9, [5, 64 * 3, 700]), (3, 5, 1000, [1, 2, 129])])
def test_prompts_and_their_completions(cuda_device, heads, kv, dim, prompts, each, shared, tails):
    Batch(*forked(prompts, each, shared, tails), heads, kv, dim, cuda_device).check()


def test_more_sequences_than_a_block_takes(cuda_device):
    # 70 sequences of 4 heads per key/value head: three blocks' rows, the last one not full
    Batch(*forked(1, 70, 640, [3, 64, 100]), 8, 2, 64, cuda_device).check()
    Batch(*forked(2, 67, 128, [0]), 16, 8, 128, cuda_device).check()


def test_nothing_shared_and_some_not(cuda_device):
    Batch(*forked(5, 1, 300, [0, 30]), 8, 2, 64, cuda_device).check()  # nobody shares
    pages, pos = forked(2, 3, 256, [9, 80])
    pages += [[500, 501, 502], [503]]  # two that share with nobody, one of them on its first token
    pos += [150, 0]
    Batch(pages, pos, 8, 2, 64, cuda_device).check()


def test_forks_of_forks(cuda_device):
    root, left, right = [40, 3], [17, 5, 21, 22], [11]
    pages = [root + left + [60], root + left + [61, 62], root + left + [63], root + right + [64], root + right + [65, 66], root + [67], [40, 68]]
    pos = [64 * 6 + 3, 64 * 7, 64 * 7 - 1, 64 * 3, 64 * 5 - 1, 64 * 2 + 9, 64 + 1]
    b = Batch(pages, pos, 32, 8, 128, cuda_device)
    plan = b.plan()
    assert len(plan.runs) == 4
    b.check(plan)


def test_long_prompts(cuda_device):
    Batch(*forked(1, 6, 64 * 300 + 5, [0, 64 * 40, 9]), 8, 2, 128, cuda_device).check()


def test_large_scores(cuda_device):
    # scores of several hundred: the running maximum moves from page to page, most weights vanish
    Batch(*forked(2, 4, 64 * 12, [1, 64 * 5 + 2]), 16, 4, 64, cuda_device, spread=8.0).check()


def test_values_and_keys_that_are_infinite_stay_so(cuda_device):
    b = Batch(*forked(1, 3, 192, [4]), 4, 2, 64, cuda_device)
    b.v[b.pages[0][1], 0, 5, 7] = float("inf")
    got = b.run(b.plan()).reshape(3, 4, 64)
    assert torch.isinf(got[:, :2, 7]).all() and torch.isfinite(got[:, 2:]).all() and torch.isfinite(got[:, :2, :7]).all()


def test_a_plan_stays_good_while_last_pages_fill(cuda_device):
    pages, pos = forked(1, 4, 256, [2, 70])
    b = Batch(pages, pos, 8, 2, 64, cuda_device)
    plan = b.plan()
    for _ in range(3):
        b.check(plan)
        b.pos = [p + 1 for p in b.pos]
        b.tok_pos += 1
        b.qkv = torch.roll(b.qkv, 1, 0) + 0.25


def test_captured_and_replayed(cuda_device):
    b = Batch(*forked(2, 4, 500, [0, 10, 100]), 32, 8, 64, cuda_device)
    plan, other = b.plan(), Batch(*forked(1, 9, 700, [0, 33]), 32, 8, 64, cuda_device, seed=3)
    plan2 = other.plan()
    want, want2 = b.check(plan).clone(), other.check(plan2).clone()
    graphs = []
    for x, p in ((b, plan), (other, plan2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.run(p)
        graphs.append(g)
    for _ in range(3):
        b.out.zero_()
        other.out.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.out, want) and torch.equal(other.out, want2)


def test_on_a_side_stream(cuda_device):
    b = Batch(*forked(2, 4, 500, [0, 10, 100]), 32, 8, 64, cuda_device)
    plan = b.plan()
    want = b.check(plan).clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(b.out)
    with torch.cuda.stream(s):
        b.run(plan, out)
    s.synchronize()
    assert torch.equal(out, want)


def test_refused(cuda_device):
    b = Batch(*forked(1, 3, 192, [4]), 4, 2, 64, cuda_device)
    plan = b.plan()
    call = lambda **c: ops.attention_decode_shared(**{**dict(qkv=b.qkv, k_off=256, v_off=384, out=b.out, n_seqs=3, n_heads=4, n_kv_heads=2, head_dim=64, scale=0.1,
                                                           tok_pos=b.tok_pos, slots=b.slots, page_table=b.table, k_cache=b.k, v_cache=b.v, plan=plan), **c})
    call()
    for change in (dict(n_seqs=2), dict(n_heads=2), dict(scale=0.0), dict(scale=-1.0), dict(k_off=450), dict(k_off=257), dict(out=b.out[:2]), dict(qkv=b.qkv.float()),
                   dict(qkv=b.qkv[:, ::2]), dict(k_cache=b.k[:, :1]), dict(page_table=b.table[:, :3].contiguous()), dict(slots=b.slots[:2]),
                   dict(tok_pos=b.tok_pos.long()), dict(v_cache=b.v.cpu())):
        with pytest.raises(ops.KernelError):
            call(**change)


def test_two_calls_at_once(cuda_device):
    a, b = Batch(*forked(2, 16, 64 * 40, [0, 300]), 32, 8, 128, cuda_device), Batch(*forked(1, 40, 64 * 30, [5, 64 * 9]), 32, 8, 128, cuda_device, seed=4)
    plans = [x.plan() for x in (a, b)]
    want = [x.check(p).clone() for x, p in zip((a, b), plans)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for x in (a, b):
            x.out.zero_()
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, x, p in zip(streams, (a, b), plans):
            with torch.cuda.stream(s):
                x.run(p)
        torch.cuda.synchronize()
        assert all(torch.equal(x.out, w) for x, w in zip((a, b), want))


def test_no_sequence(cuda_device):
    b = Batch(*forked(1, 3, 192, [4]), 4, 2, 64, cuda_device)
    plan = ops.shared_plan([], 4, 2, 64, cuda_device)
    before = b.k.clone()
    out = ops.attention_decode_shared(b.qkv[:0], 256, 384, b.out[:0], 0, 4, 2, 64, 0.1, b.tok_pos[:0], b.slots[:0], b.table, b.k, b.v, plan)
    assert out.shape == (0, 256) and torch.equal(b.k.view(torch.int16), before.view(torch.int16))


def test_a_cache_behind_the_reach_of_32_bits(cuda_device):
    # 2^31 numbers of keys and as many of values in front of the pages
    pages, pos = forked(1, 5, 64 * 3, [7, 64])
    b = Batch(pages, pos, 4, 1, 128, cuda_device)
    far = (1 << 31) // (PAGE * 128) + 3
    k, v = (torch.empty((far + b.k.shape[0], 1, PAGE, 128), dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    k[far:], v[far:] = b.k, b.v
    b.k, b.v = k, v
    b.pages = [[p + far for p in row] for row in pages]
    b.table = torch.where(b.table >= 0, b.table + far, b.table)
    got = b.run(b.plan())
    small = Batch(pages, pos, 4, 1, 128, cuda_device)
    want = small.check()
    assert torch.equal(got, want)
    assert torch.equal(k[far:].view(torch.int16), small.k.view(torch.int16)) and torch.equal(v[far:].view(torch.int16), small.v.view(torch.int16))


def test_seven_hundred_sequences(cuda_device):
    # (more heads of sequences than there are tickets for splits that meet in memory: none are needed)
    Batch(*forked(1, 700, 128, [3, 70]), 16, 16, 16, cuda_device).check()


@pytest.mark.parametrize("heads,kv,dim,prompts,each,shared,tails", [(32, 8, 64, 1, 4, 200, [40]), (32, 8, 128, 4, 8, 1000, [300, 2]), (12, 4, 80, 2, 7, 3000, [500, 0, 64])])
def test_between_products(cuda_device, heads, kv, dim, prompts, each, shared, tails):
    # recorded, every kernel may begin before the one in front has ended; the results are those of launches with a full stop in between, bit for bit
    b = Batch(*forked(prompts, each, shared, tails), heads, kv, dim, cuda_device)
    plan, n = b.plan(), prompts * each
    g = torch.Generator().manual_seed(5)
    w, w2 = ((torch.randn(s, generator=g) * 0.03).to(torch.bfloat16).to(cuda_device) for s in (((heads + 2 * kv) * dim, 512), (512, heads * dim)))
    x = torch.zeros(n, 512, dtype=torch.bfloat16, device=cuda_device)

    def run(stop):
        wait = torch.cuda.synchronize if stop else (lambda: None)
        qkv = ops.linear(x, w)
        wait()
        ops.rope_append(qkv, heads + kv, dim, dim, 0.9, b.tok_pos)
        wait()
        out = torch.empty_like(b.out)
        ops.attention_decode_shared(qkv, heads * dim, (heads + kv) * dim, out, n, heads, kv, dim, b.scale, b.tok_pos, b.slots, b.table, b.k, b.v, plan)
        wait()
        return out, ops.linear(out, w2)

    run(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [run(False) for _ in range(4)]
    for turn in range(25):
        x.copy_(torch.randn(n, 512, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        want = run(True)
        for pair in got:
            assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])
