"""Several completions of one prompt: forked sequences, shared pages and filtered sampling together, as ``generate`` uses them."""
import os

import numpy as np
import pytest
import torch

import bitnet_c_b200 as bn
import fesorax_cases
import lakadra_cases
import lotilix_cases
import mekevik_cases
import netanex_cases
import plain_llama
import rudolix_cases
from bitnet_c_b200.csrc import ops
from bitnet_c_b200.engine import ModelEngine, SeqStep, generate
from bitnet_c_b200.sampling import SamplingParams
from helpers import TOL_F32, make_model_dir, measured_bf16_bound, random_tokens, sharp_std
from tiny_configs import TINY_A, TINY_C, TINY_D, TINY_E

pytestmark = pytest.mark.gpu
LLAMAS = {"a": (TINY_A, 100), "c": (TINY_C, 300), "d": (TINY_D, 700), "e": (TINY_E, 200)}


@pytest.fixture(scope="module")
def llamas(tmp_path_factory, cuda_device):
    out = {}
    for name, (cfg, _n) in LLAMAS.items():
        for dtype in ("float32", "bfloat16"):
            d = make_model_dir(tmp_path_factory.mktemp(name + dtype), cfg, 5, dtype, matrix_std=sharp_std(cfg))
            out[name, dtype] = bn.load_model(d, dtype=dtype), plain_llama.read_model(d)
    return out


@pytest.fixture
def shared_calls(monkeypatch):
    """How often attention over shared pages was launched; it is wherever pages are shared, also where so few that it does not pay."""
    calls, real = [], ops.attention_decode_shared
    monkeypatch.setattr(ops, "shared_pays", lambda plan: bool(plan.runs))
    monkeypatch.setattr(ops, "attention_decode_shared", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    return calls


@pytest.mark.parametrize("name", sorted(LLAMAS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forks_go_on_as_sequences_of_their_own(llamas, shared_calls, name, dtype):
    model, (cfg, w) = llamas[name, dtype]
    raw, length = LLAMAS[name]
    V = raw["vocab_size"]
    prompt, other = random_tokens(1, length, V), random_tokens(2, 70, V)
    cache = model.new_cache(max_tokens=64 * 80, max_seqs=8)
    a, x = cache.open(), cache.open()
    model.step(cache, [SeqStep(a, prompt), SeqStep(x, other[:-20])])
    slots = [a, *cache.fork(a, 3)]
    own = [random_tokens(10 + i, 24, V) for i in range(6)]
    got = {s: [] for s in (*slots, x)}
    tails = dict(zip(slots, own))
    tails[x] = other[-20:] + own[5][:4]
    for t in range(12):  # forks and a stranger, one token each
        seqs = [SeqStep(s, [tails[s][t]], [0]) for s in (slots[2], x, slots[0], slots[3], slots[1])]
        logits = model.step(cache, seqs).cpu().numpy()
        for s, l in zip(seqs, logits):
            got[s.slot].append(l)
    # one of them is forked again in the middle, and one ends
    second = cache.fork(slots[1])[0]
    cache.close(slots[3])
    tails[second] = tails[slots[1]][:12] + own[4][:12]
    got[second] = list(got[slots[1]])
    for t in range(12, 24):
        seqs = [SeqStep(s, [tails[s][t]], [0]) for s in (second, slots[0], slots[1], slots[2], x)]
        logits = model.step(cache, seqs).cpu().numpy()
        for s, l in zip(seqs, logits):
            got[s.slot].append(l)
    cache.check()
    assert bool(shared_calls) == (dtype == "bfloat16")
    for s, rows in got.items():
        whole = (other[:-20] if s == x else prompt) + tails[s][:len(rows)]
        ref = plain_llama.forward(cfg, w, whole)
        tol = TOL_F32 * max(1.0, float(np.abs(ref).max())) if dtype == "float32" else measured_bf16_bound(cfg, w, whole, ref)
        off = np.abs(np.stack(rows) - ref[len(whole) - len(rows):]).max()
        assert off <= tol, (s, off, tol)


@pytest.mark.parametrize("name", ["a", "c"])
def test_completions_are_those_of_the_prompt_given_several_times(llamas, name):
    """In single precision request i draws the same tokens whether its prompt was run for it alone or forked."""
    model, _ = llamas[name, "float32"]
    V = LLAMAS[name][0]["vocab_size"]
    prompts = [random_tokens(3, 90, V), random_tokens(4, 1, V), random_tokens(5, 64, V)]
    kw = dict(temperature=0.9, top_p=0.95, seed=11, repeat_penalty=1.1, top_k=20, min_p=0.01)
    want = bn.generate(model, [p for p in prompts for _ in range(3)], 12, **kw)
    got = bn.generate(model, prompts, 12, completions=3, **kw)
    assert [c.tokens for c in got] == [c.tokens for c in want]
    assert len({tuple(c.tokens) for c in got}) > 3  # completions of one prompt differ
    again = bn.generate(model, prompts, [12, 12, 12], completions=3, max_batch=4, **kw)  # batches that cut through a prompt's completions
    assert [c.tokens for c in again] == [c.tokens for c in want]


@pytest.mark.parametrize("name", ["c", "d", "e"])
@pytest.mark.parametrize("graphs", [True, False])
def test_filtered_completions_of_shared_pages(llamas, shared_calls, name, graphs):
    """bfloat16, recorded steps and direct ones: every token is among the three that the plain model holds most probable, within rounding; one engine serves
    batches whose sequences share other pages in the same slots."""
    model, (cfg, w) = llamas[name, "bfloat16"]
    raw, length = LLAMAS[name]
    V = raw["vocab_size"]
    eng = ModelEngine(model, model.new_cache(max_tokens=64 * 90, max_seqs=6), SamplingParams(temperature=1.0, top_p=1.0, top_k=3, seed=3), use_graphs=graphs)
    prompts = [random_tokens(20, length, V), random_tokens(21, length - 7, V), random_tokens(22, length, V)]
    for some, each in (([prompts[0]], 6), (prompts[1:], 3), ([prompts[2], prompts[0], prompts[1]], 2), ([prompts[1]], 6)):
        got = generate(eng, some, 70, completions=each)
        eng.cache.check()
        assert len({tuple(c.tokens) for c in got}) == len(got)
        for i, c in enumerate(got):
            whole = some[i // each] + c.tokens[:-1]
            ref = plain_llama.forward(cfg, w, whole)
            tol = measured_bf16_bound(cfg, w, whole, ref)
            rows = ref[len(some[i // each]) - 1:]
            third = np.sort(rows, axis=1)[:, -3]
            assert all(rows[j, t] >= third[j] - 2 * tol for j, t in enumerate(c.tokens))
    assert shared_calls
    if graphs:
        assert any(key[1] for r in eng.runners.values() for key in r.graphs)  # steps with shared pages were recorded
    assert eng.cache.tokens_free() == eng.cache.max_tokens


def test_compaction_between_recorded_steps(llamas, shared_calls):
    model, _ = llamas["c", "bfloat16"]
    V = TINY_C["vocab_size"]
    got = []
    for compact in (False, True):
        cache = model.new_cache(max_tokens=64 * 60, max_seqs=6)
        eng = ModelEngine(model, cache, SamplingParams(temperature=0.9, top_k=40, seed=3))
        first = cache.open()  # something in front that goes away
        model.step(cache, [SeqStep(first, random_tokens(1, 400, V))])
        calls = []

        def emitted(i, token):
            calls.append(1)
            if compact and len(calls) == 20:
                cache.close(first)
                assert cache.compact() > 0
                cache.check()
            return False

        got.append([c.tokens for c in generate(eng, [random_tokens(2, 300, V)], 20, completions=4, callback=emitted)])
    assert got[0] == got[1]


DESIGNS = {  # the module of a design's test cases, a configuration of it and what else its weights are drawn from
    "fesorax": (fesorax_cases, fesorax_cases.CASE_A, fesorax_cases.REL_ROWS_A), "lotilix": (lotilix_cases, *lotilix_cases.CASES["A"]),
    "mekevik": (mekevik_cases, *mekevik_cases.CASES["A"]), "netanex": (netanex_cases, netanex_cases.CASES["A"]),
    "rudolix": (rudolix_cases, rudolix_cases.CASES["A"]), "lakadra": (lakadra_cases, lakadra_cases.CASES["A"]),
}


@pytest.mark.parametrize("design", sorted(DESIGNS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_other_designs_fork_their_states_and_windows(tmp_path, cuda_device, design, dtype):
    """A fork goes on as the sequence that brought the same tokens from the start: recurrent states, convolutions, latents, windows that have given pages back."""
    m, cfg, *more = DESIGNS[design]
    tensors = m.draw_weights(cfg, *more, 7)
    model = bn.load_model(m.write_folder(str(tmp_path / design), cfg, tensors), dtype=dtype)
    V = model.spec.vocab_size
    n = min(150, model.spec.max_positions - 20)
    prompt, tails = random_tokens(1, n, V), [random_tokens(2 + i, 8, V) for i in range(3)]
    cache = model.new_cache(max_tokens=64 * 40, max_seqs=8)

    def go_on(slots):
        rows = [model.step(cache, [SeqStep(s, [t[j]], [0]) for s, t in zip(slots, tails)]).cpu() for j in range(8)]
        for s in slots:
            cache.close(s)
        return torch.stack(rows)

    a = cache.open()
    model.step(cache, [SeqStep(a, prompt)])
    forked = go_on([a, *cache.fork(a, 2)])
    slots = []
    for _ in tails:
        slots.append(cache.open())
        model.step(cache, [SeqStep(slots[-1], prompt)])
    cache.check()
    alone = go_on(slots)
    # the same kernels on the same numbers: what differs is at most which page a key lies in
    assert torch.equal(forked, alone)
    assert not torch.equal(forked[-1, 0], forked[-1, 1])


def test_command_line(llamas, tmp_path, cuda_device):
    import json
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "cfg.json").write_text(json.dumps(TINY_A))
    args = [sys.executable, os.path.join(root, "bin", "bitnet"), str(tmp_path / "m"), "--random-weights", "--config", str(tmp_path / "cfg.json"), "-n", "6",
            "--prompt-token-ids", "5,17,3", "--prompt-token-ids", "9", "--temp", "0.9", "--topk", "30", "--minp", "0.01", "--completions", "3"]
    p = subprocess.run(args, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=600)
    assert p.returncode == 0, p.stderr
    lines = p.stdout.split()
    assert len(lines) == 6 and all(len(l.split(",")) <= 6 for l in lines) and len(set(lines[:3])) > 1
