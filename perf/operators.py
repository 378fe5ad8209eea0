"""The operators behind several completions of one prompt, as cases that can be timed and compared.

* ``copy``: pages of a cache copied to other pages, all planes at once: the partly filled last page of a prompt for each of its
  completions, or whole pages moved to the front of the pool.
* ``slots``: the fixed-size states of a sequence copied to the slots of its completions, all state tensors at once.
* ``attend``: attention of one new token for each of several sequences that share the pages of their prompts; the new keys
  and values go into the cache.
* ``sample``: the next token from temperature, top-k, top-p and min-p, from given random numbers.

Sizes are those of the benchmark's Llama configurations and designs, and odd ones beside them.
"""
import torch

own = False

DEVICE = "cuda:0"
PAGE = 64  # tokens per page of the cache


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # two completions of one prompt in a small model: the last page, 16 planes, latency
        dict(name="copy last page 2 forks", op="copy", planes=16, heads=8, dim=64, vdim=64, dtype="bfloat16", moves=2, rows=37, forks=True),
        # sixteen completions in the 8B sizes
        dict(name="copy last page 16 forks", op="copy", planes=32, heads=8, dim=128, vdim=128, dtype="bfloat16", moves=16, rows=51, forks=True),
        # whole pages of the 8B sizes moved to the front of the pool: the bandwidth of a copy
        dict(name="copy whole pages", op="copy", planes=32, heads=8, dim=128, vdim=128, dtype="bfloat16", moves=64, rows=64, forks=False),
        # states of a few layers whose rows are no multiple of 16 bytes, one more completion
        dict(name="slots odd rows", op="slots", tensors=12, floats=771, forks=1),
        # recurrent states of 24 layers (16 heads of 128 x 128) for seven more completions
        dict(name="slots recurrent states", op="slots", tensors=24, floats=262144, forks=7),
        # four completions of a short prompt in the 1B sizes: launches and latency
        dict(name="attend 4 of one short prompt", op="attend", prompts=1, each=4, shared=200, tail=40, heads=32, kv_heads=8, dim=64),
        # eight prompts with eight completions each, 8B sizes, prompts of unequal lengths
        dict(name="attend 8 prompts by 8", op="attend", prompts=8, each=8, shared=2048, tail=300, heads=32, kv_heads=8, dim=128),
        # many completions of one long prompt
        dict(name="attend 64 of one long prompt", op="attend", prompts=1, each=64, shared=8192, tail=500, heads=32, kv_heads=8, dim=128),
        # one sequence, the small vocabulary, top-k: latency
        dict(name="sample 1 row top-k", op="sample", rows=1, vocab=32000, dtype="float32", filters="top_k", spread=3.0),
        # a batch of 8 with a nucleus and min-p
        dict(name="sample 8 rows top-p", op="sample", rows=8, vocab=128256, dtype="float32", filters="top_p", spread=3.0),
        # many users, each with parameters of their own
        dict(name="sample 64 rows own params", op="sample", rows=64, vocab=128256, dtype="float32", filters="rows", spread=3.0),
        # a flat distribution (an early checkpoint, a high temperature) over an odd vocabulary in bfloat16: many ties, wide nuclei
        dict(name="sample 200 flat rows bf16", op="sample", rows=200, vocab=50257, dtype="bfloat16", filters="rows", spread=1.0),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["copy", "slots", "attend", "sample"])
    if op == "copy":
        heads, dim = rng.choice([(8, 64), (8, 128), (40, 128), (2, 80), (1, 192), (5, 48), (16, 96)])
        whole = rng.random() < 0.3
        case = dict(op=op, planes=_between(rng, 1, 40), heads=heads, dim=dim, vdim=rng.choice([dim, dim, 64, 0]), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]),
                    moves=_between(rng, 1, 64), rows=PAGE if whole else rng.randint(1, PAGE - 1), forks=not whole)
        # no more than the largest listed case
        while case["planes"] * case["moves"] * heads * dim * (2 if case["dtype"] == "bfloat16" else 4) > 32 * 64 * 8 * 128 * 2:
            case["moves"], case["planes"] = max(1, case["moves"] // 2), max(1, case["planes"] // 2)
        return case
    if op == "slots":
        tensors, forks = _between(rng, 1, 40), _between(rng, 1, 15)
        return dict(op=op, tensors=tensors, floats=min(_between(rng, 1, 400000), 24 * 262144 * 7 // (tensors * forks)), forks=forks)
    if op == "attend":
        heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (40, 40, 128), (6, 2, 48), (24, 1, 96), (12, 4, 80), (16, 16, 64)])
        prompts, each = _between(rng, 1, 12), _between(rng, 2, 64)
        while prompts * each > 64:
            prompts, each = max(1, prompts // 2), max(2, each - 1)
        shared = _between(rng, 1, 8192)
        while shared * prompts * kv_heads * dim > 8192 * 2 * 8 * 128:
            shared = max(1, shared // 2)
        return dict(op=op, prompts=prompts, each=each, shared=shared, tail=_between(rng, 1, 500), heads=heads, kv_heads=kv_heads, dim=dim)
    rows = _between(rng, 1, 256)
    return dict(op=op, rows=rows, vocab=min(_between(rng, 200, 262144), 64 * 128256 // rows), dtype=rng.choice(["float32", "float32", "bfloat16"]),
                filters=rng.choice(["top_k", "top_p", "min_p", "rows", "none"]), spread=rng.choice([0.3, 1.0, 3.0, 3.0]))


# ---- inputs -------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    return {"copy": _prepare_copy, "slots": _prepare_slots, "attend": _prepare_attend, "sample": _prepare_sample}[case["op"]](case, g, host)


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype) if dtype != torch.bfloat16 else torch.randn(
        shape, generator=g, device=DEVICE, dtype=torch.bfloat16)


def _prepare_copy(case, g, host):
    dtype, moves = getattr(torch, case["dtype"]), case["moves"]
    pages = 2 * moves + 3
    k = _normal((case["planes"], pages, case["heads"], PAGE, case["dim"]), dtype, g)
    v = _normal((case["planes"], pages, case["heads"], PAGE, case["vdim"]), dtype, g) if case["vdim"] else None
    order = torch.randperm(pages, generator=host).tolist()
    sources = [order[0]] * moves if case["forks"] else order[:moves]
    # (source page, page it is copied to, rows of it that are copied)
    return dict(case, k=k, v=v, list=[(s, d, case["rows"]) for s, d in zip(sources, order[moves:2 * moves])])


def _prepare_slots(case, g, host):
    slots = case["forks"] + 2
    tensors = [_normal((slots, case["floats"]), torch.float32, g) for _ in range(case["tensors"])]
    order = torch.randperm(slots, generator=host).tolist()
    state = dict(case, states=tensors, source=order[0], list=order[1:1 + case["forks"]])
    if own:  # where the states lie: a cache makes this once
        from bitnet_c_b200.csrc import ops
        state["where"] = ops.StateSlots(tensors)
    return state


def _prepare_attend(case, g, host):
    H, KV, D, B = case["heads"], case["kv_heads"], case["dim"], case["prompts"] * case["each"]
    # prompts of unequal lengths, completions at unequal places behind them
    shared = [max(1, case["shared"] - int(torch.randint(0, case["shared"] // 4 + 1, (1,), generator=host))) for _ in range(case["prompts"])]
    pos = [shared[b // case["each"]] + int(torch.randint(0, case["tail"], (1,), generator=host)) for b in range(B)]
    width = max(p // PAGE + 1 for p in pos)
    pool = case["prompts"] * (case["shared"] // PAGE + 1) + B * (case["tail"] // PAGE + 2)
    free = torch.randperm(pool, generator=host).tolist()
    rows = [[0] * width for _ in range(B)]
    for p, s in enumerate(shared):
        head = [free.pop() for _ in range(s // PAGE)]
        for b in range(p * case["each"], (p + 1) * case["each"]):
            mine = head + [free.pop() for _ in range(pos[b] // PAGE + 1 - len(head))]
            rows[b][:len(mine)] = mine
    k = _normal((pool, KV, PAGE, D), torch.bfloat16, g)
    v = _normal((pool, KV, PAGE, D), torch.bfloat16, g)
    state = dict(case, k=k, v=v, qkv=_normal((B, (H + 2 * KV) * D), torch.bfloat16, g), scale=D ** -0.5,
                 pos=torch.tensor(pos, dtype=torch.int32, device=DEVICE), slots=torch.arange(B, dtype=torch.int32, device=DEVICE),
                 table=torch.tensor(rows, dtype=torch.int32, device=DEVICE), out=torch.empty((B, H * D), dtype=torch.bfloat16, device=DEVICE),
                 longest=max(pos) + 1)
    if own:  # which sequences share which pages: follows the page tables alone, made when a sequence takes a new page
        from bitnet_c_b200.csrc import ops
        state["plan"] = ops.shared_plan([r[:p // PAGE + 1] for r, p in zip(rows, pos)], H, KV, D, DEVICE)
    return state


def _prepare_sample(case, g, host):
    n, V = case["rows"], case["vocab"]
    logits = torch.randn((n, V), generator=g, device=DEVICE) * case["spread"]
    if case["spread"] >= 3.0:  # a model that knows some: a few tokens stand out
        at = torch.randint(0, V, (n, 24), generator=g, device=DEVICE)
        logits.scatter_add_(1, at, 9.0 + 2.5 * torch.randn((n, 24), generator=g, device=DEVICE))
    rand = lambda: torch.rand(n, generator=g, device=DEVICE)  # noqa: E731
    given = {"top_k": (0.8, 50, 1.0, 0.0), "top_p": (0.7, 0, 0.9, 0.02), "min_p": (1.0, 0, 1.0, 0.05), "none": (1.0, 0, 1.0, 0.0)}.get(case["filters"])
    if given is None:  # every row has parameters of its own, some of them switched off
        given = (0.3 + rand(), torch.where(rand() < 0.5, (rand() * 200).int(), 0).int(), torch.where(rand() < 0.7, 0.5 + 0.5 * rand(), 1.0),
                 torch.where(rand() < 0.3, 0.1 * rand(), 0.0))
    return dict(case, logits=logits.to(getattr(torch, case["dtype"])), given=given, u=rand())


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    return {"copy": _run_copy, "slots": _run_slots, "attend": _run_attend, "sample": _run_sample}[state["op"]](state)


def _run_copy(s):
    k, v = s["k"], s["v"]
    if own:
        from bitnet_c_b200.csrc import ops
        ops.copy_pages(k, v, s["list"])
    else:
        src, dst, _rows = torch.tensor(s["list"], device=DEVICE).unbind(1)
        k[:, dst, :, :s["rows"]] = k[:, src, :, :s["rows"]]
        if v is not None:
            v[:, dst, :, :s["rows"]] = v[:, src, :, :s["rows"]]
    return [k, v]


def _run_slots(s):
    if own:
        from bitnet_c_b200.csrc import ops
        ops.copy_slots(s["where"], s["source"], s["list"])
    else:
        to = torch.tensor(s["list"], device=DEVICE)
        for t in s["states"]:
            t[to] = t[s["source"]].clone()
    return s["states"]


def _run_attend(s):
    B, H, KV, D = s["prompts"] * s["each"], s["heads"], s["kv_heads"], s["dim"]
    if own:
        from bitnet_c_b200.csrc import ops
        ops.attention_decode_shared(s["qkv"], H * D, (H + KV) * D, s["out"], B, H, KV, D, s["scale"], s["pos"], s["slots"], s["table"],
                                    s["k"], s["v"], s["longest"], s["plan"])
        return s["out"], s["k"], s["v"]
    pos = s["pos"].long()
    q, new_k, new_v = s["qkv"].split([H * D, KV * D, KV * D], 1)
    at = s["table"].long()[torch.arange(B, device=DEVICE), pos // PAGE]
    s["k"][at, :, pos % PAGE] = new_k.reshape(B, KV, D)
    s["v"][at, :, pos % PAGE] = new_v.reshape(B, KV, D)
    seen = lambda c: c[s["table"].long()].float().transpose(1, 2).reshape(B, KV, -1, D)  # noqa: E731  [sequence, head, position, number]
    scores = torch.matmul(q.float().reshape(B, KV, H // KV, D), seen(s["k"]).transpose(2, 3)) * s["scale"]
    hidden = torch.arange(scores.shape[3], device=DEVICE)[None, :] > pos[:, None]
    scores = scores.masked_fill(hidden[:, None, None], float("-inf"))
    w = (scores - scores.amax(3, keepdim=True)).exp()
    values = seen(s["v"]).masked_fill(hidden[:, None, :, None], 0.0)
    out = torch.matmul(w, values) / w.sum(3, keepdim=True)
    return out.reshape(B, H * D).to(torch.bfloat16), s["k"], s["v"]


def _run_sample(s):
    temperature, top_k, top_p, min_p = s["given"]
    if own:
        from bitnet_c_b200.csrc import ops
        return ops.sample_filtered(s["logits"], temperature, top_k, top_p, min_p, u=s["u"])
    n, V = s["logits"].shape
    column = lambda x: torch.as_tensor(x, device=DEVICE).expand(n).double()[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p, u = (column(x) for x in (temperature, top_k, top_p, min_p, s["u"]))
    value, token = s["logits"].float().sort(dim=1, descending=True, stable=True)  # equal ones: the lower index first
    value = value.double()
    w = ((value - value[:, :1]) / temperature).exp()  # sums in 64 bits: a running sum lies next to a border often enough
    place = torch.arange(V, device=DEVICE)[None, :]
    kept = (place < top_k) | (top_k <= 0)
    w = torch.where(kept, w, 0.0)
    below = w.cumsum(1) - w
    kept &= (below <= top_p * w.sum(1, keepdim=True)) | (top_p <= 0) | (top_p >= 1)
    kept &= w >= min_p
    w = torch.where(kept, w, 0.0)
    running = w.cumsum(1)
    passed = (running > u * running[:, -1:]) & kept
    chosen = torch.where(passed.any(1), passed.int().argmax(1), kept.sum(1) - 1)
    return token.gather(1, chosen[:, None])[:, 0].int()


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    if case["op"] == "copy":
        item = 2 if case["dtype"] == "bfloat16" else 4
        once = case["planes"] * case["heads"] * case["rows"] * (case["dim"] + case["vdim"]) * item
        return {"bytes": once * (case["moves"] + (1 if case["forks"] else case["moves"])), "flops": 0}
    if case["op"] == "slots":
        return {"bytes": case["tensors"] * case["floats"] * 4 * (case["forks"] + 1), "flops": 0}
    if case["op"] == "attend":
        # lengths are drawn: the mean of each
        H, KV, D, B = case["heads"], case["kv_heads"], case["dim"], case["prompts"] * case["each"]
        shared, tail = case["shared"] * 7 / 8, case["tail"] / 2
        keys = case["prompts"] * shared + B * tail
        return {"bytes": keys * KV * D * 4 + B * (2 * H + 4 * KV) * D * 2, "flops": 4 * H * D * B * (shared + tail)}
    item = 2 if case["dtype"] == "bfloat16" else 4
    return {"bytes": case["rows"] * (case["vocab"] * item + 8), "flops": 4 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"copy": _exact_copy, "slots": _exact_slots, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _exact_copy(s):
    for tensor in (s["k"], s["v"]):
        if tensor is not None:
            for src, dst, rows in s["list"]:  # sources are never written
                tensor[:, dst, :, :rows].copy_(tensor[:, src, :, :rows].clone())
    return [s["k"], s["v"]]


def _exact_slots(s):
    for tensor in s["states"]:
        for slot in s["list"]:
            tensor[slot].copy_(tensor[s["source"]].clone())
    return s["states"]


def _exact_attend(s):
    H, KV, D = s["heads"], s["kv_heads"], s["dim"]
    out = torch.empty((s["qkv"].shape[0], H, D), dtype=torch.float64, device=DEVICE)
    table, pos = s["table"].tolist(), s["pos"].tolist()
    for b, p in enumerate(pos):
        row = s["qkv"][b].reshape(H + 2 * KV, D)
        s["k"][table[b][p // PAGE], :, p % PAGE] = row[H:H + KV]
        s["v"][table[b][p // PAGE], :, p % PAGE] = row[H + KV:]
    for b, p in enumerate(pos):
        pages = table[b][:p // PAGE + 1]
        keys = torch.cat([s["k"][i] for i in pages], 1)[:, :p + 1].double()
        values = torch.cat([s["v"][i] for i in pages], 1)[:, :p + 1].double()
        q = s["qkv"][b, :H * D].double().reshape(KV, H // KV, D)
        out[b] = torch.einsum("ghp,gpd->ghd", torch.softmax(torch.einsum("ghd,gpd->ghp", q, keys) * s["scale"], 2), values).reshape(H, D)
    return out.reshape(-1, H * D), s["k"], s["v"]


def _exact_sample(s):
    import bisect
    import itertools

    n = s["logits"].shape[0]
    parameters = [torch.as_tensor(x).expand(n).tolist() for x in (*s["given"], s["u"])]  # in single precision, as the operator takes them
    token = []
    for row, (temperature, top_k, top_p, min_p, u) in zip(s["logits"].double().cpu(), zip(*parameters)):
        order = torch.argsort(-row, stable=True)
        w = torch.exp((row[order] - row[order[0]]) / temperature)[:top_k if top_k > 0 else None].tolist()
        if 0 < top_p < 1:
            running = list(itertools.accumulate(w))
            w = w[:bisect.bisect_right(running, top_p * running[-1]) + 1]
        while w[-1] < min_p:
            w.pop()
        running = list(itertools.accumulate(w))
        token.append(int(order[min(bisect.bisect_right(running, u * running[-1]), len(w) - 1)]))
    return torch.tensor(token, dtype=torch.int32)
