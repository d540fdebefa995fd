"""Beam search over a paged key-value cache, operator by operator, as cases that can be timed and compared.

* ``attend``   attention of one new token of every sequence over its pages (``paged.paged_attention``);
* ``fork``     sequences that go on as copies of others, or end: full pages are shared, a page that is not full is copied
               (``paged.fork_pages``);
* ``compact``  the pages in use moved to the front of the pool (``paged.compact_pages``);
* ``select``   the best continuations of every group of beams over beams and vocabulary (``beam.beam_select``);
* ``reorder``  the recurrent states and convolution histories of beams put in the order of their parents (``beam.reorder_states``).

Lengths, tables and parents go by the case alone (its ``structure``), the values in them by the seed.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 151936             # of the NVFP4 model
REC = (32, 128, 128)       # its recurrent state of a layer: value heads, key width, value width
CONV = (8192, 3)           # its convolution history of a layer: channels, taps but one


def listed():
    return [
        # one user behind a short prompt: latency
        {"name": "attend_1x100", "op": "attend", "batch": 1, "shortest": 100, "longest": 100, "heads": 16, "kv_heads": 2, "dim": 256, "page": 16,
         "type": "bf16", "gate": True, "window": 0, "sinks": 0, "structure": 1},
        # a small server: sequences of all lengths, one of them without a token yet
        {"name": "attend_32x8192", "op": "attend", "batch": 32, "shortest": 0, "longest": 8192, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64,
         "type": "bf16", "gate": True, "window": 0, "sinks": 0, "structure": 2},
        # a few long documents, many heads
        {"name": "attend_4x131072", "op": "attend", "batch": 4, "shortest": 100001, "longest": 131072, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128,
         "type": "bf16", "gate": False, "window": 0, "sinks": 0, "structure": 3},
        # streams that see their last tokens and the first few, checked in fp32
        {"name": "attend_48x20000_window_fp32", "op": "attend", "batch": 48, "shortest": 1, "longest": 20000, "heads": 16, "kv_heads": 4, "dim": 64, "page": 24,
         "type": "fp32", "gate": False, "window": 1024, "sinks": 4, "structure": 4},
        # one request of four beams: latency
        {"name": "fork_1x4", "op": "fork", "groups": 1, "beams": 4, "shortest": 203, "longest": 203, "layers": 2, "kv_heads": 2, "dim": 256, "page": 16,
         "type": "bf16", "spare": 0.3, "ended": 0, "structure": 5},
        # a server of sixteen requests of eight beams, all attention layers of the 48-layer model, two requests have ended
        {"name": "fork_16x8", "op": "fork", "groups": 16, "beams": 8, "shortest": 300, "longest": 2100, "layers": 12, "kv_heads": 2, "dim": 256, "page": 64,
         "type": "bf16", "spare": 0.1, "ended": 2, "structure": 6},
        # small pages of a pool that a few requests hold
        {"name": "compact_7", "op": "compact", "groups": 7, "beams": 1, "shortest": 5, "longest": 700, "layers": 1, "kv_heads": 2, "dim": 256, "page": 16,
         "type": "bf16", "spare": 0.6, "ended": 0, "structure": 7},
        # a pool whose requests have mostly ended, before the rest of it is given back
        {"name": "compact_40", "op": "compact", "groups": 40, "beams": 1, "shortest": 100, "longest": 2500, "layers": 12, "kv_heads": 2, "dim": 256, "page": 64,
         "type": "bf16", "spare": 1.0, "ended": 0, "structure": 8},
        # one request of four beams: latency
        {"name": "select_1x4", "op": "select", "batch": 1, "beams": 4, "vocab": VOCAB, "type": "bf16", "ended": 0.25, "structure": 9},
        # a server of 32 requests of eight beams, fp32 logits
        {"name": "select_32x8_fp32", "op": "select", "batch": 32, "beams": 8, "vocab": VOCAB, "type": "fp32", "ended": 0.1, "structure": 10},
        # one request of four beams, the three recurrent layers of a group of four
        {"name": "reorder_1x4", "op": "reorder", "groups": 1, "beams": 4, "layers": 3, "structure": 11},
        # eight requests of eight beams, a third of the 48-layer model's recurrent layers
        {"name": "reorder_8x8", "op": "reorder", "groups": 8, "beams": 8, "layers": 12, "structure": 12},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm, odd ones among them."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op, structure = rng.choice(["attend", "attend", "attend", "fork", "compact", "select", "select", "reorder"]), rng.randrange(1 << 30)
    kind = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    page = rng.choice([1, 7, 8, 16, 16, 24, 32, 64, 64, 100, 128, 256])
    if op == "attend":
        heads, kv_heads, dim = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (32, 8, 128), (16, 4, 64), (8, 8, 128), (12, 4, 96), (7, 1, 80),
                                           (20, 5, 64), (48, 2, 128), (5, 5, 40), (64, 1, 192), (32, 1, 256)])
        batch = _log(rng, 1, 200)
        room = (1 << 30) // (batch * kv_heads * dim * (4 if kind == "fp32" else 2))            # positions: half of the largest listed case's bytes
        longest = _log(rng, 1, min(131072, room))
        window = rng.random() < 0.3
        return {"op": op, "batch": batch, "shortest": rng.choice([0, 0, 1, longest // 2, longest]), "longest": longest, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "page": page, "type": kind, "gate": rng.random() < 0.5, "window": _log(rng, 1, 4096) if window else 0,
                "sinks": rng.choice([0, 1, 4, 5, 64]) if window else 0, "structure": structure}
    if op in ("fork", "compact"):
        kv_heads, dim = rng.choice([(2, 256), (2, 256), (8, 128), (4, 64), (1, 80), (5, 40)])
        beams, layers = rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), rng.choice([1, 2, 3, 8, 12])
        row = beams * layers * kv_heads * dim * (4 if kind == "fp32" else 2) * 2
        groups = _log(rng, 1, max(1, min(40, (1 << 30) // (row * page))))
        room = (1 << 30) // (groups * row)
        longest = _log(rng, 1, max(1, min(8192, room)))
        return {"op": op, "groups": groups, "beams": beams, "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest, "layers": layers,
                "kv_heads": kv_heads, "dim": dim, "page": page, "type": kind, "spare": rng.choice([0.1, 0.3, 1.0, 2.0]),
                "ended": rng.randint(0, groups // 2), "structure": structure}
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        return {"op": op, "batch": min(_log(rng, 1, 64), 256 // beams), "beams": beams, "vocab": _log(rng, 40, 262144), "type": rng.choice(["bf16", "fp32"]),
                "ended": rng.choice([0, 0, 0.1, 0.5]), "structure": structure}
    beams = rng.choice([2, 3, 4, 5, 8, 12, 16])
    return {"op": op, "groups": _log(rng, 1, 64 // beams), "beams": beams, "layers": rng.choice([1, 3, 3, 6, 12]), "structure": structure}


# --------------------------------------------------------------------------------- what the cases look like
def _lengths(case, count):
    """Lengths spread evenly between the shortest and the longest, in no order; both occur where there are two."""
    r = np.random.RandomState(case["structure"])
    n = r.randint(case["shortest"], case["longest"] + 1, count)
    n[0] = case["longest"]
    n[-1] = case["shortest"] if count > 1 else n[-1]
    return r.permutation(n).astype(np.int32)


def _attend_table(case):
    """(lengths, table, pages of the pool): every sequence's pages lie anywhere, entries behind its last one are -1."""
    n, page = _lengths(case, case["batch"]), case["page"]
    held = -(-n // page)
    width, total = max(1, int(held.max())), int(held.sum())
    r = np.random.RandomState(case["structure"] + 1)
    place = r.permutation(total + 3)[:total]
    table = np.full((case["batch"], width), -1, np.int32)
    table[np.arange(width)[None] < held[:, None]] = place
    return n, table, total + 3


def _visible(case, n):
    return n if not case["window"] else np.minimum(n, case["sinks"] + case["window"])


def _parents(case, groups, beams, ended):
    """Of every beam: the beam that it continues, in its own group.  A beam that goes on stays in its place; -1: its request has ended."""
    r = np.random.RandomState(case["structure"] + 2)
    stays = r.rand(groups, beams) < 0.6
    stays[np.arange(groups), r.randint(0, beams, groups)] = True
    pick = np.argmax(stays[:, None, :] * (1 + r.rand(groups, beams, beams)), axis=2)
    parents = np.where(stays, np.arange(beams)[None], pick) + beams * np.arange(groups)[:, None]
    parents[r.permutation(groups)[:ended]] = -1
    return parents.reshape(-1).astype(np.int32)


def _fork_table(case):
    """(lengths, table, reference counts, parents): beams of a group have the same length and share nine tenths of their full pages."""
    groups, beams, page = case["groups"], case["beams"], case["page"]
    n = np.repeat(_lengths(case, groups), beams)
    held, shared = -(-n // page), (n // page * 9) // 10 if beams > 1 else n * 0
    width = max(1, int(held.max())) + 1
    r = np.random.RandomState(case["structure"] + 1)
    first = np.arange(groups * beams) // beams * beams
    columns = np.arange(width)[None]
    inside = columns < held[:, None]
    lender = np.where(columns < shared[:, None], first[:, None], np.arange(groups * beams)[:, None])
    used, number = np.unique((lender * width + columns)[inside], return_inverse=True)
    pages = len(used) + groups * beams + int(case["spare"] * len(used))
    place = r.permutation(pages)[:len(used)]
    table = np.full((groups * beams, width), -1, np.int32)
    table[inside] = place[number.reshape(-1)]
    refs = np.bincount(table[inside], minlength=pages).astype(np.int32)
    return n.astype(np.int32), table, refs, _parents(case, groups, beams, case["ended"] if case["op"] == "fork" else 0)


def _generator(seed, salt):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 64 + salt)
    return g


def _normal(seed, salt, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=_generator(seed, salt), device=DEVICE, dtype=F32) * std).to(dtype)


def _on_device(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)


def prepare(case, seed):
    s, op = {"case": case}, case["op"]
    if op == "attend":
        n, table, pages = _attend_table(case)
        kind, shape = TYPES[case["type"]], (pages, case["page"], case["kv_heads"], case["dim"])
        # scores of a standard deviation of 2: some positions count, most do not
        s.update(q=_normal(seed, 1, case["batch"], case["heads"], case["dim"], std=2.0, dtype=kind), k=_normal(seed, 2, *shape, dtype=kind),
                 v=_normal(seed, 3, *shape, dtype=kind), table=_on_device(table), lengths=_on_device(n), gate=None)
        if case["gate"]:
            s["gate"] = _normal(seed, 4, case["batch"], case["heads"], case["dim"], dtype=kind)
        return s
    if op in ("fork", "compact"):
        n, table, refs, parents = _fork_table(case)
        shape = (len(refs), case["layers"], case["page"], case["kv_heads"], case["dim"])
        s.update(k=_normal(seed, 1, *shape, dtype=TYPES[case["type"]]), v=_normal(seed, 2, *shape, dtype=TYPES[case["type"]]), table=_on_device(table),
                 lengths=_on_device(n), refs=_on_device(refs), parents=_on_device(parents))
        return s
    if op == "select":
        batch, beams, r = case["batch"], case["beams"], np.random.RandomState(case["structure"])
        s["logits"] = _normal(seed, 1, batch, beams, case["vocab"], std=3.0, dtype=TYPES[case["type"]])
        # log-probabilities of some twenty tokens; one request is at its first token, of which all beams but one say nothing
        s["scores"] = torch.randn((batch, beams), generator=_generator(seed, 2), device=DEVICE, dtype=F32) * 2.0 - 40.0
        if batch > 1:
            s["scores"][-1, 1:] = -math.inf
        s["finished"] = _on_device(r.rand(batch, beams) < case["ended"])
        s["eos"] = int(r.randint(0, case["vocab"]))
        return s
    count = case["groups"] * case["beams"]
    s["rec"] = _normal(seed, 1, count, case["layers"], *REC, std=0.1, dtype=F32)
    s["conv"] = _normal(seed, 2, count, case["layers"], *CONV)
    s["parents"] = _on_device(_parents(case, case["groups"], case["beams"], 0))
    return s


# --------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from quickdraw_b200 import beam, paged
        if op == "attend":
            return paged.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], gate=s["gate"], window=case["window"], sinks=case["sinks"])
        if op == "fork":
            table, lengths, refs = paged.fork_pages(s["k"], s["v"], s["table"], s["lengths"], s["refs"], s["parents"])
            return {"table": table, "lengths": lengths, "refs": refs, "k": s["k"], "v": s["v"]}
        if op == "compact":
            table, refs, used = paged.compact_pages(s["k"], s["v"], s["table"], s["refs"])
            return {"table": table, "refs": refs, "used": used, "k": s["k"], "v": s["v"]}
        if op == "select":
            scores, parents, tokens = beam.beam_select(s["logits"], s["scores"], finished=s["finished"], eos=s["eos"])
            return {"scores": scores, "parents": parents, "tokens": tokens}
        beam.reorder_states([s["rec"], s["conv"]], s["parents"])
        return {"rec": s["rec"], "conv": s["conv"]}
    if op == "attend":
        return _attend(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["gate"], case["window"], case["sinks"])
    if op == "fork":
        table, lengths, refs = _fork(s["k"], s["v"], s["table"], s["lengths"], s["refs"], s["parents"])
        return {"table": table, "lengths": lengths, "refs": refs, "k": s["k"], "v": s["v"]}
    if op == "compact":
        table, refs, used = _compact(s["k"], s["v"], s["table"], s["refs"])
        return {"table": table, "refs": refs, "used": used, "k": s["k"], "v": s["v"]}
    if op == "select":
        scores, parents, tokens = _select(s["logits"], s["scores"], s["finished"], s["eos"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    s["rec"].copy_(s["rec"][s["parents"].long()])
    s["conv"].copy_(s["conv"][s["parents"].long()])
    return {"rec": s["rec"], "conv": s["conv"]}


def _attend(q, k, v, table, lengths, gate, window, sinks):
    """softmax(q k / sqrt(dim)) v over what each sequence sees; rows that see nothing are zeros."""
    page, n = k.shape[1], lengths.long()[:, None]
    room = table.shape[1] * page
    i = torch.arange(min(room, sinks + window) if window else room, device=q.device)[None]          # the i-th position that is seen
    position = torch.where((i >= sinks) & (n > sinks + window), i + n - sinks - window, i) if window else i.expand(q.shape[0], -1)
    seen = position < n
    position = torch.where(seen, position, 0)
    pages = table.long().gather(1, position // page).clamp(min=0)
    batch, heads, dim = q.shape
    kv_heads = k.shape[2]
    keys = k[pages, position % page].float()                                                        # [batch, seen, kv_heads, dim]
    scores = torch.einsum("bhgd,bnhd->bhgn", q.float().view(batch, kv_heads, heads // kv_heads, dim), keys) / math.sqrt(dim)
    del keys
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(dim=-1, keepdim=True)
    values = torch.where(seen[:, :, None, None], v[pages, position % page].float(), 0.0)
    out = torch.einsum("bhgn,bnhd->bhgd", weights / torch.where(total == 0, 1.0, total), values).reshape(batch, heads, dim)
    if gate is not None:
        out = out / (1 + torch.exp(-gate.float()))
    return out.to(q.dtype)


def _fork(k, v, table, lengths, refs, parents):
    """Sequence b goes on as a copy of sequence parents[b] (-1: it ends); one that is its own parent stays as it is.  The page that is not full goes to the
    parent itself or else to its first copy; the others, in order, get the lowest free pages and a copy of its rows."""
    count, width = table.shape
    page, pages = k.shape[2], refs.numel()
    here, columns = torch.arange(count, device=table.device), torch.arange(width, device=table.device)[None]
    parent, stays = parents.long().clamp(min=0), parents == here
    n = torch.where(parents >= 0, lengths[parent], 0)
    full, rest = (n // page).long(), n % page
    first = torch.full((count,), count, device=table.device).scatter_reduce(0, parent, torch.where(stays, -1, torch.where(parents >= 0, here, count)), "amin")
    takes = (parents >= 0) & ((first[parent] == here) | stays)
    needs = (rest > 0) & (parents >= 0) & ~takes
    kept = (columns < full[:, None]) | ((columns == full[:, None]) & ((rest > 0) & takes)[:, None])
    new = torch.where(stays[:, None], table, torch.where(kept, table[parent], -1))
    counted = refs.clone()
    counted.index_add_(0, table.clamp(min=0).reshape(-1).long(), -(table >= 0).reshape(-1).int())
    counted.index_add_(0, new.clamp(min=0).reshape(-1).long(), (new >= 0).reshape(-1).int())
    free = torch.argsort(counted > 0, stable=True)                                                 # free pages first, each kind in order
    who = needs.nonzero()[:, 0]
    to, source = free[:who.numel()], table[parent[who], full[who]].long()
    new[who, full[who]] = to.int()
    counted[to] = 1
    rows = (torch.arange(page, device=table.device)[None] < rest[who][:, None])[:, None, :, None, None]
    k[to] = torch.where(rows, k[source], k[to])
    v[to] = torch.where(rows, v[source], v[to])
    return new, n, counted


def _compact(k, v, table, refs):
    """Pages in use behind the first `used` ones move, in order, to the free ones in front; pages that are not used any more keep what they hold."""
    taken = refs > 0
    used, number = taken.sum(), torch.arange(refs.numel(), device=refs.device)
    source, to = (taken & (number >= used)).nonzero()[:, 0], (~taken & (number < used)).nonzero()[:, 0]
    k[to], v[to] = k[source], v[source]
    place, counted = number.int(), refs.clone()
    place[source] = to.int()
    counted[to], counted[source] = refs[source], 0
    return torch.where(table >= 0, place[table.clamp(min=0).long()], table), counted, used.int()


def _select(logits, scores, finished, eos):
    """The best `beams` sums of a score and a log-probability; among equals the lowest beam and token.  A finished beam has one continuation, `eos`, at no cost.  A
    beam's best continuation takes the beam's place, the others the places left, in order.  64 bits: sums of different beams lie next to one another."""
    batch, beams, vocab = logits.shape
    x = logits.double()
    top = x.amax(dim=-1, keepdim=True)
    each = x - (top + torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True)))
    ends = torch.where(torch.arange(vocab, device=x.device) == eos, 0.0, -math.inf).double()
    total = scores.double()[:, :, None] + torch.where(finished[:, :, None], ends, each)
    total = torch.where(torch.isnan(total), -math.inf, total).reshape(batch, beams * vocab)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :beams], at[:, :beams]
    parent, token = at // vocab, at % vocab
    same = parent[:, :, None] == torch.arange(beams, device=x.device)
    leads = (same & (same.long().cumsum(1) == 1)).any(2)                                            # [batch, rank]: the first of its parent
    left = torch.argsort(same.any(1).long(), dim=1, stable=True)                                    # places without a continuation of their own first
    place = torch.where(leads, parent, left.gather(1, ((~leads).long().cumsum(1) - 1).clamp(min=0)))
    put = lambda t: torch.empty_like(t).scatter_(1, place, t)  # noqa: E731
    return put(best).float(), put(parent + beams * torch.arange(batch, device=x.device)[:, None]).int(), put(token)


# --------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, size = case["op"], 4 if case.get("type") == "fp32" else 2
    if op == "attend":
        n = _visible(case, _attend_table(case)[0])
        seen, rows = int(n.sum()), case["batch"] * case["heads"] * case["dim"]
        return {"bytes": 2 * seen * case["kv_heads"] * case["dim"] * size + rows * size * (3 if case["gate"] else 2) + 4 * (int((-(-n // case["page"])).sum()) + case["batch"]),
                "flops": 4 * seen * case["heads"] * case["dim"]}
    if op in ("fork", "compact"):
        n, table, refs, parents = _fork_table(case)
        row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
        if op == "fork":
            here = np.arange(len(n))
            moved = int((n[parents] % case["page"])[(parents >= 0) & (parents != here)].sum())
        else:
            moved = int((refs[int((refs > 0).sum()):] > 0).sum()) * case["page"]
        return {"bytes": 2 * moved * row + 8 * (table.size + refs.size) + 8 * n.size, "flops": 0}
    if op == "select":
        count = case["batch"] * case["beams"]
        return {"bytes": count * case["vocab"] * size + 21 * count, "flops": 3 * count * case["vocab"]}
    parents = _parents(case, case["groups"], case["beams"], 0)
    moved = parents != np.arange(len(parents))
    row = case["layers"] * (4 * int(np.prod(REC)) + 2 * int(np.prod(CONV)))
    return {"bytes": (int(moved.sum()) + len(np.unique(parents[moved]))) * row, "flops": 0}


# --------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    op = case["op"]
    if op == "attend":
        s = prepare(case, seed)
        n, table, _ = _attend_table(case)
        batch, heads, dim, kv_heads = case["batch"], case["heads"], case["dim"], case["kv_heads"]
        out = torch.zeros((batch, heads, dim), dtype=F64, device=DEVICE)
        for b in range(batch):
            p = np.arange(n[b])
            if case["window"]:
                p = p[(p < case["sinks"]) | (p >= n[b] - case["window"])]
            if not len(p):
                continue
            pages, rows = _on_device(table[b][p // case["page"]].astype(np.int64)), _on_device(p % case["page"])
            for h in range(kv_heads):
                mine = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
                keys, values = s["k"][pages, rows, h].to(F64), s["v"][pages, rows, h].to(F64)
                out[b, mine] = torch.softmax(s["q"][b, mine].to(F64) @ keys.T * dim ** -0.5, dim=1) @ values
        return out * torch.sigmoid(s["gate"].to(F64)) if case["gate"] else out
    if op == "select":
        s = prepare(case, seed)
        batch, beams, vocab = s["logits"].shape
        scores = torch.empty((batch, beams), dtype=F64, device=DEVICE)
        for b in range(batch):
            found = []
            for i in range(beams):
                if bool(s["finished"][b, i]):
                    found.append((float(s["scores"][b, i]), i))
                else:
                    found += [(t, i) for t in (torch.log_softmax(s["logits"][b, i].to(F64), 0).topk(min(beams, vocab)).values + s["scores"][b, i].to(F64)).tolist()]
            found = sorted((f for f in found if f[0] > -math.inf), key=lambda f: -f[0])[:beams]
            if len(found) < beams:
                return None                                   # too few continuations: ties at minus infinity decide
            places = [None] * beams
            for t, i in found:                                # a beam's best in the beam's place, the others in what is left
                if places[i] is None:
                    places[i] = t
            leads, rest = {(t, i) for i, t in enumerate(places) if t is not None}, iter([i for i in range(beams) if places[i] is None])
            for t, i in found:
                if (t, i) in leads:
                    leads.remove((t, i))
                else:
                    places[next(rest)] = t
            scores[b] = torch.tensor(places, dtype=F64)
        return {"scores": scores, "parents": None, "tokens": None}
    return None                                               # moved, not computed
