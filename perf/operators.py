"""What the operators of serving several continuations of a prompt from little memory are measured on: linears whose weights are 4-bit
codes with group scales (``ops/int4.py``), and pages of a key-value cache that sequences share, copy, pack and give back on the device
(``ops/pages.py``).

  linear     one linear of a decoder layer: ``rows`` rows of activations, a packed weight matrix, with the norm ahead of it, the residual
             behind it or the gated unit that the layer has there. A weight is ``scale[n, k // group] * (code[n, k] - zero[n, k // group])``
  quantise   a bf16 weight matrix to 4 bits and the values that it then stands for, as a program does when it opens a checkpoint
  turn       ``children`` continuations of a prompt in slot 0: they are forked off it, get pages for ``new`` tokens each, are drawn again
             with repeats (some end, some go on twice) and are given back
  swap       two sequences of a full pool, one after the other: copied to a second pool, given back, the pool compacted; then they get pages
             again and are copied back

Weights are N(0, 0.02), as models are initialised, in the types that checkpoints hold; activations are N(0, 1) with gains of 1 + N(0, 0.1),
a few columns ten times as large, as residual streams have them. Caches hold any bits: they are copied. Lengths end inside a page and at
its end."""
from __future__ import annotations

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
EPS = 1e-6
NORM_ROWS = 8            # up to so many rows a linear takes the norm ahead of it


def listed():
    return [
        # the output projection of a small model's layer, one user: nothing but latency
        dict(name="output 1 row", kind="linear", rows=1, n=1024, k=1024, group=128, zeros=False, gated=False, norm=False, residual=True, seed=0),
        # a matrix that no tile divides, with zero points and small groups, a few sequences
        dict(name="odd 3 rows", kind="linear", rows=3, n=2741, k=2056, group=32, zeros=True, gated=False, norm=True, residual=False, seed=0),
        # the gated half of a wide feed-forward, one user
        dict(name="gate up 1 row", kind="linear", rows=1, n=16384, k=4096, group=128, zeros=False, gated=True, norm=True, residual=False, seed=0),
        # its other half, a few users, as checkpoints with zero points have it
        dict(name="down 8 rows", kind="linear", rows=8, n=4096, k=16384, group=64, zeros=True, gated=False, norm=False, residual=True, seed=0),
        # the packed projection of queries, keys and values: a batch of users, of no round number
        dict(name="qkv 203 rows", kind="linear", rows=203, n=6144, k=4096, group=128, zeros=False, gated=False, norm=False, residual=False, seed=0),
        # a long prompt through the wide gated half
        dict(name="gate up 4096 rows", kind="linear", rows=4096, n=16384, k=4096, group=128, zeros=True, gated=True, norm=False, residual=False, seed=0),
        # a small model's matrix
        dict(name="quantise 1024 x 4096", kind="quantise", n=1024, k=4096, group=128, zeros=False, gated=False, seed=0),
        # a wide feed-forward's packed matrix, with zero points
        dict(name="quantise 32768 x 4096", kind="quantise", n=16384, k=4096, group=64, zeros=True, gated=True, seed=0),
        # four continuations of a short prompt, a small model
        dict(name="turn 4 of 300", kind="turn", children=4, length=300, new=20, layers=12, width=1024, page=16, seed=0),
        # a wide tree over a long document
        dict(name="turn 64 of 30011", kind="turn", children=64, length=30011, new=130, layers=12, width=512, page=16, seed=0),
        # a few short sequences
        dict(name="swap 200 of 4", kind="swap", slots=4, length=200, layers=12, width=512, page=16, seed=0),
        # a full pool of long ones
        dict(name="swap 4090 of 8", kind="swap", slots=8, length=4090, layers=12, width=512, page=16, seed=0),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "quantise", "turn", "swap"))
    seed = rng.randrange(1 << 20)
    if kind in ("linear", "quantise"):
        gated = rng.random() < 0.4
        c = dict(kind=kind, n=_log(rng, 64, 16384), k=_log(rng, 32, 2048) * 8, group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.5, gated=gated, seed=seed)
        if kind == "quantise":
            return {**c, "k": min(c["k"], 4096)}
        rows = _log(rng, 1, 4096) if rng.random() < 0.5 else rng.randint(1, 24)
        while rows * c["n"] * (1 + gated) * c["k"] > 4096 * 32768 * 4096:
            rows //= 2
        return {**c, "rows": rows, "norm": rows <= NORM_ROWS and rng.random() < 0.5, "residual": not gated and rng.random() < 0.5}
    page = rng.choice((8, 16, 32, 64))
    c = dict(kind=kind, layers=rng.randint(2, 24), width=8 * _log(rng, 8, 128), page=page, seed=seed)
    if kind == "turn":
        return {**c, "children": _log(rng, 1, 64), "length": _log(rng, 1, 20000), "new": _log(rng, 1, 200)}
    return {**c, "slots": rng.randint(2, 8), "length": _log(rng, 2, 2000)}


# -- 4-bit weights ----------------------------------------------------------------------------------------------------------
def _generator(case, seed):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["seed"])


def _by_group(w, group):
    """[N, K] as [N, groups, group], the last group filled up with zeros."""
    n, k = w.shape
    return torch.nn.functional.pad(w, (0, -k % group)).view(n, -1, group)


def _quantised(w, group, zeros):
    """Codes [N, K], scales [N, groups] in bf16 and zero points [N, groups] of ``w``."""
    f = _by_group(w.float(), group)
    if zeros:
        low, high = f.amin(-1).clamp(max=0), f.amax(-1).clamp(min=0)
        scale = ((high - low) / 15).to(BF16)
    else:
        scale = (f.abs().amax(-1) / 7).to(BF16)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    s = scale.float()
    zero = (torch.round(-low / s) if zeros else torch.full_like(s, 8)).clamp(0, 15)
    code = (torch.round(f / s[..., None]) + zero[..., None]).clamp(0, 15)
    return code.view(w.shape[0], -1)[:, :w.shape[1]].to(torch.uint8).contiguous(), scale, zero.to(torch.uint8)


def _values(code, scale, zero, group):
    c = _by_group(code.float(), group)
    return ((c - zero.float()[..., None]) * scale.float()[..., None]).view(code.shape[0], -1)[:, :code.shape[1]]


def _prepare_linear(case, seed):
    g = _generator(case, seed)
    t, k, rows_w = case["rows"], case["k"], case["n"] * (1 + case["gated"])
    x = torch.randn(t, k, generator=g, device="cuda")
    x[:, torch.randint(0, k, (max(1, k // 512),), generator=g, device="cuda")] *= 10
    w = (torch.randn(rows_w, k, generator=g, device="cuda") * 0.02).to(BF16)
    code, scale, zero = _quantised(w, case["group"], case["zeros"])
    gain = (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(BF16)
    residual = torch.randn(t, case["n"], generator=g, device="cuda").to(BF16)
    s = dict(case=case, x=x.to(BF16), gain=gain if case["norm"] else None, residual=residual if case["residual"] else None)
    if own:        # a program lays its weights out once
        from ironpangu_b200.ops import int4

        s["weight"] = int4.pack(code, scale, zero if case["zeros"] else None, group=case["group"], gated=case["gated"])
    else:
        s.update(code=code, scale=scale, zero=zero)
    return s


def _run_linear(s):
    c = s["case"]
    if own:
        from ironpangu_b200.ops import int4

        return int4.linear(s["x"], s["weight"], norm_w=s["gain"], eps=EPS, residual=s["residual"])
    x = s["x"].float()
    if c["norm"]:
        # the norm is an operator of its own, whose rows are bf16
        x = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["gain"].float()).to(BF16).float()
    y = x @ _values(s["code"], s["scale"], s["zero"], c["group"]).T
    if c["gated"]:
        gate, up = y[:, :c["n"]], y[:, c["n"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(BF16)


def _exact_linear(case, seed):
    s = _prepare_linear(case, seed)
    n, k, group = case["n"], case["k"], case["group"]
    x = s["x"].to(F64)
    if case["norm"]:
        x = (x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / k + EPS) * s["gain"].to(F64)).to(BF16).to(F64)
    at = torch.arange(k, device="cuda") // group

    def product(lo, hi):
        w = (s["code"][lo:hi].to(F64) - s["zero"][lo:hi].to(F64)[:, at]) * s["scale"][lo:hi].to(F64)[:, at]
        return torch.einsum("tk,nk->tn", x, w)

    y = product(0, n)
    if case["gated"]:
        y = y * torch.sigmoid(y) * product(n, 2 * n)
    return y + s["residual"].to(F64) if case["residual"] else y


def _weight_bytes(case):
    groups = -(-case["k"] // case["group"])
    return case["n"] * (1 + case["gated"]) * (case["k"] / 2 + groups * (3 if case["zeros"] else 2))


def _prepare_quantise(case, seed):
    w = torch.randn(case["n"] * (1 + case["gated"]), case["k"], generator=_generator(case, seed), device="cuda") * 0.02
    return dict(case=case, w=w.to(BF16))


def _run_quantise(s):
    c = s["case"]
    if own:
        from ironpangu_b200.ops import int4

        return int4.quantise(s["w"], group=c["group"], zeros=c["zeros"], gated=c["gated"]).dequantise()
    return _values(*_quantised(s["w"], c["group"], c["zeros"]), c["group"]).to(BF16)


def _exact_quantise(case, seed):
    w, group = _prepare_quantise(case, seed)["w"].to(F64), case["group"]
    at = torch.arange(case["k"], device="cuda") // group
    spread = lambda v: v[:, at]
    empty = torch.zeros(w.shape[0], int(at[-1]) + 1, dtype=F64, device="cuda")
    top = empty.scatter_reduce(1, at.expand_as(w), w, "amax")            # zero is among the values
    low = empty.scatter_reduce(1, at.expand_as(w), w, "amin")
    s = ((top - low) / 15 if case["zeros"] else torch.maximum(top, -low) / 7).to(F32).to(BF16).to(F64)
    s = torch.where(s == 0, 1.0, s)
    z = torch.round(-low / s).clamp(0, 15) if case["zeros"] else torch.full_like(s, 8)
    q = (torch.round(w / spread(s)) + spread(z)).clamp(0, 15)
    return (q - spread(z)) * spread(s)


# -- pages ------------------------------------------------------------------------------------------------------------------
# Plain form: `s` holds table [slots, most pages of one], lengths [slots], refs [pages] and caches [layers' keys and values, pages, rows, width]
def _free_pages(refs):
    return torch.argsort((refs > 0).to(torch.uint8), stable=True)           # the free ones first, lowest first


def _count(entries, pages):
    return torch.zeros(pages + 1, dtype=I32, device="cuda").index_add_(0, torch.where(entries < 0, pages, entries).reshape(-1).long(),
                                                                       torch.ones(entries.numel(), dtype=I32, device="cuda"))[:pages]


def _extend(s, slots, tokens):
    page, at = s["page"], torch.arange(s["table"].shape[1], device="cuda")[None]
    have, want = (-(-v.long() // page) for v in (s["lengths"][slots], tokens))
    new = (at >= have[:, None]) & (at < want[:, None])
    order = torch.cumsum(new.reshape(-1).long(), 0).view_as(new) - 1
    fresh = _free_pages(s["refs"])[order.clamp(min=0)].to(I32)
    rows = torch.where(new, fresh, s["table"][slots])
    s["refs"] += _count(torch.where(new, fresh, -1), s["refs"].numel())
    s["table"][slots] = rows
    s["lengths"][slots] = torch.maximum(s["lengths"][slots], tokens)


def _fork(s, src, dst):
    page, n = s["page"], src.numel()
    rows, lengths = s["table"][src], s["lengths"][src]
    replaced = (src[:, None] == dst[None]).any(1)
    earlier = ((src[:, None] == src[None]) & (torch.arange(n, device="cuda")[None] < torch.arange(n, device="cuda")[:, None])).any(1)
    used = lengths % page
    copies = (used > 0) & (earlier | ~replaced)
    s["table"][dst] = rows
    s["lengths"][dst] = lengths
    s["refs"].copy_(_count(s["table"], s["refs"].numel()))
    last = (lengths // page).long().clamp(max=rows.shape[1] - 1)
    old = rows.gather(1, last[:, None])[:, 0]
    fresh = _free_pages(s["refs"])[(torch.cumsum(copies.long(), 0) - 1).clamp(min=0)].to(I32)
    new = torch.where(copies, fresh, old)
    at, to = old[copies].long(), new[copies].long()
    live = torch.arange(page, device="cuda")[None] < used[copies][:, None]
    s["caches"][:, to] = torch.where(live[None, :, :, None], s["caches"][:, at], s["caches"][:, to])
    s["table"][dst, last] = torch.where(used > 0, new, s["table"][dst, last])
    s["refs"].copy_(_count(s["table"], s["refs"].numel()))


def _release(s, slots):
    s["table"][slots] = -1
    s["lengths"][slots] = 0
    s["refs"].copy_(_count(s["table"], s["refs"].numel()))


def _compact(s):
    live = s["refs"] > 0
    pages = torch.arange(live.numel(), device="cuda")
    moves = live & (pages >= live.sum())
    at = moves.nonzero()[:, 0]
    to = _free_pages(s["refs"])[:at.numel()]
    s["caches"][:, to] = s["caches"][:, at]
    where = pages.clone()
    where[at] = to
    s["refs"][to] = s["refs"][at]
    s["refs"][at] = 0
    s["table"].copy_(torch.where(s["table"] < 0, s["table"], where[s["table"].clamp(min=0).long()].to(I32)))


def _copy(src, dst, at, to, rows):
    live = torch.arange(src.shape[2], device="cuda")[None] < rows[:, None]
    at, to = at.long(), to.long()
    dst[:, to] = torch.where(live[None, :, :, None], src[:, at], dst[:, to])


def _caches(g, case, pages):
    return torch.randint(-32768, 32767, (2 * case["layers"], pages, case["page"], case["width"]), generator=g, device="cuda", dtype=torch.int16).view(BF16)


def _pages_of(tokens, page):
    return -(-tokens // page)


def _empty_pool(g, case, slots, most, pages):
    s = dict(case=case, page=case["page"], table=torch.full((slots, most), -1, dtype=I32, device="cuda"), lengths=torch.zeros(slots, dtype=I32, device="cuda"),
             refs=torch.zeros(pages, dtype=I32, device="cuda"), caches=_caches(g, case, pages))
    if own:
        from ironpangu_b200.ops import pages as P

        s["pool"] = P.PagePool(list(s["caches"].unbind(0)), slots=slots, max_pages=most)
        s.update(table=s["pool"].table, lengths=s["pool"].lengths, refs=s["pool"].refs)
    return s


def _start(s, slots, tokens):
    s["pool"].extend(slots, tokens) if own else _extend(s, slots.long(), tokens)


def _prepare_turn(case, seed):
    g = _generator(case, seed)
    n, length, new, page = case["children"], case["length"], case["new"], case["page"]
    most = _pages_of(length + new, page)
    pages = _pages_of(length, page) + n * (_pages_of(new, page) + 2) + 7
    s = _empty_pool(g, case, n + 1, most, pages)
    zero = torch.zeros(1, dtype=I32, device="cuda")
    _start(s, zero, zero + length)
    s.update(prompt=torch.zeros(n, dtype=I32, device="cuda"), children=torch.arange(1, n + 1, dtype=I32, device="cuda"),
             tokens=length + torch.randint(1, new + 1, (n,), generator=g, device="cuda", dtype=I32),
             parents=torch.randint(1, n + 1, (n,), generator=g, device="cuda", dtype=I32))
    return s


def _bits(caches):
    return caches.view(torch.int16)


def _run_turn(s):
    if own:
        p = s["pool"]
        p.fork(s["prompt"], s["children"])
        p.extend(s["children"], s["tokens"])
        p.fork(s["parents"], s["children"])
        drawn = p.table.clone(), p.lengths.clone(), p.refs.clone()
        p.free(s["children"])
    else:
        children, parents = s["children"].long(), s["parents"].long()
        _fork(s, s["prompt"].long(), children)
        _extend(s, children, s["tokens"])
        _fork(s, parents, children)
        drawn = s["table"].clone(), s["lengths"].clone(), s["refs"].clone()
        _release(s, children)
    return {"drawn": drawn, "table": s["table"], "lengths": s["lengths"], "refs": s["refs"], "caches": _bits(s["caches"])}


def _prepare_swap(case, seed):
    g = _generator(case, seed)
    n, page = case["slots"], case["page"]
    most = _pages_of(case["length"], page)
    s = _empty_pool(g, case, n, most, n * most + 5)
    lengths = (torch.rand(n, generator=g, device="cuda") * 0.1 + 0.9) * case["length"]
    lengths = lengths.ceil().to(I32)
    _start(s, torch.arange(n, dtype=I32, device="cuda"), lengths)
    counts = [_pages_of(int(v), page) for v in lengths]
    s.update(store=_caches(g, case, most + 3), ids=torch.arange(2, most + 2, dtype=I32, device="cuda"), going=[])
    if own:
        from ironpangu_b200.ops import pages as P

        s["store_set"] = P.PageSet(list(s["store"].unbind(0)))
    for i in (0, n - 1):
        rows = (int(lengths[i]) - page * torch.arange(counts[i], device="cuda")).clamp(max=page).to(I32)
        s["going"].append((torch.tensor([i], dtype=I32, device="cuda"), i, lengths[i:i + 1].clone(), counts[i], rows))
    return s


def _run_swap(s):
    for slot, i, tokens, count, rows in s["going"]:
        ids = s["ids"][:count]
        if own:
            from ironpangu_b200.ops import pages as P

            p = s["pool"]
            P.copy(p.pages, s["store_set"], p.table[i, :count], ids, rows)
            p.free(slot)
            p.compact()
            p.extend(slot, tokens)
            P.copy(s["store_set"], p.pages, ids, p.table[i, :count], rows)
        else:
            at = slot.long()
            _copy(s["caches"], s["store"], s["table"][i, :count], ids, rows)
            _release(s, at)
            _compact(s)
            _extend(s, at, tokens)
            _copy(s["store"], s["caches"], ids, s["table"][i, :count], rows)
    return {"table": s["table"], "lengths": s["lengths"], "refs": s["refs"], "caches": _bits(s["caches"]), "store": _bits(s["store"])}


# -- what the measurement calls ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    return {"linear": _prepare_linear, "quantise": _prepare_quantise, "turn": _prepare_turn, "swap": _prepare_swap}[case["kind"]](case, seed)


def run(state):
    return {"linear": _run_linear, "quantise": _run_quantise, "turn": _run_turn, "swap": _run_swap}[state["case"]["kind"]](state)


def exact(case, seed):
    if case["kind"] == "linear":
        return _exact_linear(case, seed)
    return _exact_quantise(case, seed) if case["kind"] == "quantise" else None           # pages are copied


def work(case):
    if case["kind"] == "linear":
        t, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": _weight_bytes(case) + 2 * t * (k + n * (1 + case["residual"])) + 2 * k * case["norm"], "flops": 2 * t * n * (1 + case["gated"]) * k}
    if case["kind"] == "quantise":
        values = case["n"] * (1 + case["gated"]) * case["k"]
        return {"bytes": 4 * values + 2 * _weight_bytes(case), "flops": 6 * values}
    row = 2 * case["layers"] * case["width"] * 2                # bytes of one position in all caches
    page, length = case["page"], case["length"]
    if case["kind"] == "turn":
        # the partly filled page of the prompt for every child, about the same again for two of five children drawn again (those drawn twice); the
        # rows of the table that fork, extend, fork and free read and write
        n, pages = case["children"], _pages_of(length + case["new"] // 2, page)
        return {"bytes": 2 * row * n * (length % page + 0.4 * page / 2) + 4 * n * pages * 6, "flops": 0}
    # out, into the holes, back
    return {"bytes": 2 * 3 * 2 * 0.95 * length * row, "flops": 0}
