"""What the operators of a decode step of many continuations are measured on: attention for rows that share a long prefix, whose keys and
values are read once for all of them (``ops/shared_prefix.py``), and sampling over the whole vocabulary from given random numbers
(``ops/sampling.py``).

  attend   ``sequences`` sequences in ``groups`` groups; the sequences of a group share a prefix of up to ``prefix`` positions, and each has up
           to ``own`` positions of its own behind it. The last ``each`` positions of every sequence are query rows: one for a decode step,
           more for questions that are asked of one document. A row sees the positions up to its own. Keys and values lie in pages
  sample   one token for each of ``rows`` rows of logits: those are kept that ``cut`` says, and the one is drawn at which the kept tokens'
           weights, added up by rising ids, pass the row's random number

Queries and keys are N(0, 1) with keys of a common mean, so that scores are as uneven as trained heads have them, values N(0, 1) with a mean
per column; pages lie anywhere in the pool. Logits are N(0, 2) with some tokens far ahead, as language models give them; temperatures lie
around 1."""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def listed():
    return [
        # two continuations of a short prompt, a small model: nothing but latency
        dict(name="attend 2 of 500", kind="attend", sequences=2, each=1, groups=1, prefix=500, own=40, heads=8, kv=4, dim=128, page=16, seed=0),
        # a handful, narrow heads, no round number anywhere
        dict(name="attend 5 of 1111", kind="attend", sequences=5, each=1, groups=1, prefix=1111, own=70, heads=8, kv=2, dim=64, page=16, seed=0),
        # a few continuations of an ordinary prompt, the 2B model's heads
        dict(name="attend 8 of 4000", kind="attend", sequences=8, each=1, groups=1, prefix=4000, own=300, heads=16, kv=4, dim=128, page=16, seed=0),
        # users of three system prompts in one step
        dict(name="attend 27 of 3 x 9001", kind="attend", sequences=27, each=1, groups=3, prefix=9001, own=900, heads=16, kv=4, dim=128, page=16, seed=0),
        # many continuations of a long document, the wide model's heads
        dict(name="attend 64 of 30011", kind="attend", sequences=64, each=1, groups=1, prefix=30011, own=500, heads=32, kv=8, dim=128, page=16, seed=0),
        # eight questions of 128 tokens about a long document, as prompts
        dict(name="attend 8 x 128 of 16384", kind="attend", sequences=8, each=128, groups=1, prefix=16384, own=128, heads=32, kv=8, dim=128, page=16, seed=0),
        # one user of a small model
        dict(name="sample 1 of 32000", kind="sample", rows=1, vocab=32000, dtype="f32", cut="top_p", seed=0),
        # one user, the sampling defaults of a server
        dict(name="sample 1 of 151936", kind="sample", rows=1, vocab=151936, dtype="f32", cut="top_k", seed=0),
        # a few users, weak tokens left out
        dict(name="sample 8 of 128000", kind="sample", rows=8, vocab=128000, dtype="f32", cut="min_p", seed=0),
        # a batch of requests, each with its own wishes
        dict(name="sample 27 of 151936", kind="sample", rows=27, vocab=151936, dtype="f32", cut="mixed", seed=0),
        # continuations that are drawn from the whole distribution
        dict(name="sample 64 of 151936", kind="sample", rows=64, vocab=151936, dtype="f32", cut="none", seed=0),
        # a full server with logits as a bf16 product leaves them, in which many are equal
        dict(name="sample 256 of 128000 bf16", kind="sample", rows=256, vocab=128000, dtype="bf16", cut="top_p", seed=0),
    ]


HEADS = ((8, 4, 128), (16, 4, 128), (32, 8, 128), (32, 4, 128), (8, 2, 64), (16, 16, 64), (14, 2, 64), (12, 2, 128))
CUTS = ("none", "top_k", "top_p", "min_p", "mixed")


def _log(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    seed = rng.randrange(1 << 20)
    if rng.random() < 0.5:
        return dict(kind="sample", rows=_log(rng, 1, 256), vocab=_log(rng, 100, 151936), dtype=rng.choice(("f32", "f32", "bf16")), cut=rng.choice(CUTS), seed=seed)
    heads, kv, dim = rng.choice(HEADS)
    case = dict(kind="attend", sequences=_log(rng, 1, 64), each=1 if rng.random() < 0.7 else _log(rng, 2, 128), groups=1, prefix=_log(rng, 1, 30000), own=_log(rng, 1, 800),
                heads=heads, kv=kv, dim=dim, page=rng.choice((8, 16, 32, 64)), seed=seed)
    case["own"] = max(case["own"], case["each"])
    case["groups"] = rng.randint(1, min(4, case["sequences"]))
    while case["sequences"] * case["each"] * (case["prefix"] + case["own"]) * heads * dim > 1024 * 16512 * 32 * 128 or case["sequences"] * case["each"] > 1024:
        case["each"] = max(1, case["each"] // 2)
    return case


def _generator(case, seed):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["seed"])


# -- attention ---------------------------------------------------------------------------------------------------------------
def _shape(case):
    """Sequences of each group, its shared positions, and every sequence's own positions: a matter of the case, not of the inputs."""
    g = torch.Generator().manual_seed(case["seed"] * 7919 + 13)
    n, groups = case["sequences"], case["groups"]
    cuts = sorted((torch.randperm(n - 1, generator=g)[:groups - 1] + 1).tolist())
    counts = [b - a for a, b in zip([0] + cuts, cuts + [n])]
    shared = [case["prefix"]] + [max(1, round(case["prefix"] * f)) for f in (torch.rand(groups - 1, generator=g) * 0.8 + 0.2).tolist()]
    mine = torch.randint(case["each"], case["own"] + 1, (n,), generator=g).tolist()
    return counts, shared, mine


def _prepare_attend(case, seed):
    g = _generator(case, seed)
    counts, shared, mine = _shape(case)
    n, each, page, hk, d = case["sequences"], case["each"], case["page"], case["kv"], case["dim"]
    whole = [s // page for s in shared]                                  # pages that a group's sequences have in common
    prefix_of = [s for c, s in zip(counts, shared) for _ in range(c)]
    lengths = [s + m for s, m in zip(prefix_of, mine)]
    most = max(-(-v // page) for v in lengths + shared)
    table, taken = [], 0
    fronts = []
    for s, w in zip(shared, whole):                                      # the group's slot: its prompt's pages
        fronts.append(list(range(taken, taken + -(-s // page))))
        taken += -(-s // page)
    for i, (c, w) in enumerate(zip(counts, whole)):
        for _ in range(c):
            length = lengths[len(table)]
            fresh = -(-length // page) - w
            table.append(fronts[i][:w] + list(range(taken, taken + fresh)))
            taken += fresh
    table += fronts
    pages = taken + 3
    where = torch.randperm(pages, generator=g, device="cuda").to(I32)
    ids = torch.tensor([r + [-1] * (most - len(r)) for r in table], device="cuda")
    table = torch.where(ids < 0, -1, where[ids.clamp(min=0)]).to(I32).contiguous()
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    k = (randn(pages, page, hk, d) + randn(hk, d) * 0.5).to(BF16)
    v = (randn(pages, page, hk, d) + randn(hk, d) * 0.5).to(BF16)
    for i, (s, c) in enumerate(zip(shared, counts)):                     # a partly filled page of the prefix is each sequence's own, with the same rows
        if s % page:
            at, to = table[n + i, s // page].long(), table[sum(counts[:i]):sum(counts[:i + 1]), s // page].long()
            for cache in (k, v):
                cache[to, :s % page] = cache[at, :s % page]
    last = torch.tensor(lengths, device="cuda")
    positions = (last[:, None] - each + torch.arange(each, device="cuda")[None]).reshape(-1).to(I32)
    slots = torch.arange(n, device="cuda").repeat_interleave(each).to(I32)
    groups = torch.tensor([[sum(counts[:i]) * each, c * each, s, n + i] for i, (c, s) in enumerate(zip(counts, shared))], dtype=I32, device="cuda")
    q = randn(n * each, case["heads"] * d).to(BF16)
    return dict(case=case, q=q, k=k, v=v, positions=positions, slots=slots, table=table, groups=groups)


def _rows_of(cache, table, positions, page):
    """What lies at the positions ``[..., n]`` of the slots whose table rows are ``[..., pages]``: ``[..., n, kv heads, dim]``."""
    at = table.long().gather(-1, positions // page) * page + positions % page
    return cache.view(-1, *cache.shape[2:])[at]


def _run_attend(s):
    c = s["case"]
    h, hk, d, page = c["heads"], c["kv"], c["dim"], c["page"]
    if own:
        from ironpangu_b200.ops import shared_prefix

        return shared_prefix.attention(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["table"], s["groups"], heads=h, kv_heads=hk, head_dim=d, scale=d ** -0.5)
    counts, shared, mine = _shape(c)
    each, outs, first = c["each"], [], 0
    for i, (count, n) in enumerate(zip(counts, shared)):
        sl = slice(first * each, (first + count) * each)
        q = s["q"][sl].float().view(-1, hk, h // hk, d)
        everyone = torch.arange(n, device="cuda")
        behind = n + torch.arange(max(mine[first:first + count]), device="cuda")
        # the sequences' own positions: the same for all rows of a sequence
        own_at = behind[None].expand(count, -1).clamp(max=s["table"].shape[1] * page - 1)
        table = s["table"][first:first + count]
        hidden = behind[None] > s["positions"][sl].long()[:, None]
        prefix_k, prefix_v = (_rows_of(x, s["table"][len(mine) + i], everyone, page).float() for x in (s["k"], s["v"]))
        own_k, own_v = (_rows_of(x, table.clamp(min=0), own_at, page).float() for x in (s["k"], s["v"]))
        by_sequence = q.view(count, each, hk, h // hk, d)
        own_scores = torch.einsum("sekgd,sjkd->sekgj", by_sequence, own_k).flatten(0, 1).masked_fill(hidden[:, None, None], -math.inf)
        scores = torch.cat([torch.einsum("tkgd,jkd->tkgj", q, prefix_k), own_scores], -1) * d ** -0.5
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        total = weights.sum(-1, keepdim=True)
        out = torch.einsum("tkgj,jkd->tkgd", weights[..., :n], prefix_v)
        out += torch.einsum("sekgj,sjkd->sekgd", weights[..., n:].view(count, each, hk, h // hk, -1), own_v).flatten(0, 1)
        outs.append((out / total).reshape(-1, h * d))
        first += count
    return torch.cat(outs).to(BF16)


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    h, hk, d, page, each = case["heads"], case["kv"], case["dim"], case["page"], case["each"]
    out = torch.empty(s["q"].shape, dtype=F64, device="cuda")
    groups = s["groups"].tolist()
    positions, table = s["positions"].tolist(), s["table"].long()
    for first, rows, n, slot in groups:
        for r in range(first, first + rows, each):                       # a sequence
            length = positions[r + each - 1] + 1
            at = torch.arange(length, device="cuda")
            pages = torch.where(at < n, table[slot][(at // page).clamp(max=table.shape[1] - 1)], table[r // each][at // page])
            visible = at[None] <= s["positions"][r:r + each].long()[:, None]
            for j in range(hk):
                k, v = (x[pages, at % page, j].to(F64) for x in (s["k"], s["v"]))
                for i in range(j * (h // hk), (j + 1) * (h // hk)):
                    z = s["q"][r:r + each, i * d:(i + 1) * d].to(F64) @ k.T / math.sqrt(d)
                    out[r:r + each, i * d:(i + 1) * d] = torch.softmax(torch.where(visible, z, -math.inf), 1) @ v
    return out


def _work_attend(case):
    counts, shared, mine = _shape(case)
    each, row = case["each"], 2 * 2 * case["kv"] * case["dim"]           # bytes of a position's key and value
    prefix_of = [s for c, s in zip(counts, shared) for _ in range(c)]
    seen = sum(each * (p + m) - each * (each - 1) // 2 for p, m in zip(prefix_of, mine))
    return {"bytes": row * (sum(shared) + sum(mine)) + 2 * 2 * len(mine) * each * case["heads"] * case["dim"], "flops": 4 * seen * case["heads"] * case["dim"]}


# -- sampling ----------------------------------------------------------------------------------------------------------------
def _prepare_sample(case, seed):
    g = _generator(case, seed)
    t, v = case["rows"], case["vocab"]
    logits = torch.randn(t, v, generator=g, device="cuda") * 2
    likely = torch.randint(0, v, (t, 20), generator=g, device="cuda")
    logits.scatter_add_(1, likely, torch.rand(t, 20, generator=g, device="cuda") * 10 + 4)
    rand = lambda: torch.rand(t, generator=g, device="cuda")
    pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (t,), generator=g, device="cuda")]
    s = dict(case=case, logits=logits.to(BF16) if case["dtype"] == "bf16" else logits, uniforms=rand(), inv_temperature=1 / (0.6 + 0.8 * rand()), top_k=None, top_p=None, min_p=None)
    cut = case["cut"]
    if cut in ("top_k", "mixed"):
        s["top_k"] = (torch.exp(rand() * math.log(1000)).to(I32) if cut == "mixed" else pick([20, 40, 50])).to(I32)
    if cut in ("top_p", "mixed"):
        s["top_p"] = 0.5 + 0.49 * rand()
    if cut in ("min_p", "mixed"):
        s["min_p"] = pick([0.02, 0.05, 0.1])
    if cut == "mixed":                                                   # who asks for what; greedy rows among them
        s["top_k"] = torch.where(rand() < 0.5, s["top_k"], 0).to(I32)
        s["top_p"] = torch.where(rand() < 0.5, s["top_p"], 1.0)
        s["min_p"] = torch.where(rand() < 0.3, s["min_p"], 0.0)
        s["inv_temperature"] = torch.where(rand() < 0.15, 0.0, s["inv_temperature"])
    return s


def _run_sample(s):
    if own:
        from ironpangu_b200.ops import sampling

        ids, probs = sampling.sample(s["logits"], s["uniforms"], inv_temperature=s["inv_temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], probs=True)
        return {"ids": ids, "probs": probs}
    # in 64 bits: the sums decide between tokens
    t, v = s["logits"].shape
    greedy = (s["inv_temperature"] <= 0)[:, None]
    z = s["logits"].double() * torch.where(greedy, 1.0, s["inv_temperature"].double()[:, None])
    weights = torch.exp(z - z.amax(1, keepdim=True))
    falling, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    ranked = weights.gather(1, order)
    place = torch.arange(v, device="cuda")[None]
    kept = torch.ones_like(ranked, dtype=torch.bool)
    if s["top_k"] is not None:
        k = torch.where((s["top_k"] < 1) | (s["top_k"] > v), v, s["top_k"])
        kept &= place < k[:, None]
    if s["min_p"] is not None:
        kept &= ranked >= s["min_p"].double()[:, None]
    if s["top_p"] is not None:
        mass = torch.where(kept, ranked, 0.0)
        ahead = torch.cumsum(mass, 1) - mass
        kept &= (ahead < s["top_p"].double()[:, None] * mass.sum(1, keepdim=True)) | (s["top_p"] >= 1)[:, None]
    kept = (kept & ~greedy) | (place == 0)
    mass = torch.zeros_like(weights).scatter_(1, order, torch.where(kept, ranked, 0.0))      # by rising ids
    cumulative = torch.cumsum(mass, 1)
    total = cumulative[:, -1:]
    past = (cumulative > s["uniforms"].double()[:, None] * total) & (mass > 0)
    ids = torch.where(past.any(1), past.to(torch.uint8).argmax(1), torch.where(mass > 0, place, 0).amax(1))
    return {"ids": ids.to(I32), "probs": (mass.gather(1, ids[:, None]) / total)[:, 0].float()}


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    found = []
    for r in range(case["rows"]):
        x = s["logits"][r].to(F64)
        it = float(s["inv_temperature"][r])
        if it <= 0:
            found.append(1.0)
            continue
        order = torch.argsort(-x, stable=True)
        p = torch.softmax(x * it, 0)
        n = x.numel()
        if s["top_k"] is not None and 0 < int(s["top_k"][r]) < n:
            n = int(s["top_k"][r])
        if s["min_p"] is not None:
            n = min(n, max(1, int((p >= p.max() * float(s["min_p"][r])).sum())))
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            run = torch.cumsum(p[order[:n]], 0)
            n = min(n, max(1, int((run[:-1] < run[-1] * float(s["top_p"][r])).sum()) + 1))
        ids = order[:n].sort().values
        run = torch.cumsum(p[ids], 0)
        at = min(n - 1, int((run <= run[-1] * float(s["uniforms"][r])).sum()))
        found.append(float(p[ids[at]] / run[-1]))
    return {"ids": None, "probs": torch.tensor(found, dtype=F64, device="cuda")}


# -- what the measurement calls ----------------------------------------------------------------------------------------------
def prepare(case, seed):
    return _prepare_attend(case, seed) if case["kind"] == "attend" else _prepare_sample(case, seed)


def run(state):
    return _run_attend(state) if state["case"]["kind"] == "attend" else _run_sample(state)


def exact(case, seed):
    return _exact_attend(case, seed) if case["kind"] == "attend" else _exact_sample(case, seed)


def work(case):
    if case["kind"] == "attend":
        return _work_attend(case)
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": case["rows"] * (case["vocab"] * size + 8), "flops": 4 * case["rows"] * case["vocab"]}
