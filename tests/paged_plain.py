"""Plain 64-bit forms of the paged cache's operators and of beam selection, a sequence at a time on the CPU, and data for them."""

import math

import torch

F64 = torch.float64


def visible(n, window, sinks):
    return [p for p in range(n) if not window or p < sinks or p >= n - window]


def attention(q, k, v, table, lengths, scale=None, gate=None, window=0, sinks=0):
    """(out, bound): softmax over what is seen, in 64 bits, and how far a result of 32-bit sums may be from it.

    The bound: a score is a sum of dim products in 32 bits, off by at most dim * 2^-24 * scale * |q| |k| (plus 2^-22 of itself for the scale, the
    difference and the exponential's argument in base 2, and 2^-22 for the exponential), so a weight is off by that relative to itself and a
    weighted mean by twice that of the largest |v|; a weight in two bf16 pieces adds 2^-16, the sums over n rows n * 2^-24 at most, of which the
    running ones of a tile, a warp and a part make far fewer (32 + n / 64 are counted).  Then half a step of the result's type."""
    q, k, v, table, lengths = (t.cpu() for t in (q, k, v, table, lengths))
    gate = None if gate is None else gate.cpu()
    batch, heads, dim = q.shape
    pages, page, kv_heads, _ = k.shape
    scale = dim ** -0.5 if scale is None else scale
    out, bound = torch.zeros((batch, heads, dim), dtype=F64), torch.zeros((batch, heads, dim), dtype=F64)
    step = torch.finfo(q.dtype).eps / 2
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        rows = [(int(table[b, p // page]), p % page) for p in visible(n, window, sinks)]
        rows = [(i, r) for i, r in rows if 0 <= i < pages]
        if not rows:
            continue
        at = torch.tensor([i for i, _ in rows]), torch.tensor([r for _, r in rows])
        for h in range(heads):
            keys, values = k[at[0], at[1], h // (heads // kv_heads)].to(F64), v[at[0], at[1], h // (heads // kv_heads)].to(F64)
            x = keys @ q[b, h].to(F64) * scale
            top = x.max()
            if top == -math.inf:
                continue
            w = torch.exp(x - top)
            out[b, h] = (w @ values) / w.sum()
            delta = dim * 2 ** -24 * abs(scale) * float(q[b, h].to(F64).norm() * keys.norm(dim=1).max()) + 2 ** -22 * float(x.abs().max() + 1)
            bound[b, h] = (2 * delta + 2 ** -16 + (32 + len(rows) / 64) * 2 ** -24) * values.abs().max()
    if gate is not None:
        g = torch.sigmoid(gate.to(F64))
        out, bound = out * g, bound * g + out.abs() * g * 2 ** -21
    return out, bound + step * (out.abs() + bound)


def cache(lengths, page, layers, kv_heads, dim, dtype, seed, spare=3, shared=0, width=None, device="cuda"):
    """(k, v, table, lengths, refs): sequences of these lengths over pages in no order; the first `shared` full pages are those of the first sequence.
    Rows that belong to nobody hold NaN."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    ids, table = 0, torch.full((len(lengths), max(1, width or max(held))), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for j in range(held[b]):
            if b and j < min(shared, n // page, lengths[0] // page):
                table[b, j] = table[0, j]
            else:
                table[b, j], ids = ids, ids + 1
    pages = ids + spare
    place = torch.randperm(pages, generator=g).int()
    table = torch.where(table >= 0, place[table.clamp(min=0).long()], table)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    pools = []
    for _ in range(2):
        pool = torch.randn((pages, layers, page, kv_heads, dim), generator=g)
        owned = torch.zeros((pages, page), dtype=torch.bool)
        for b, n in enumerate(lengths):
            for p in range(n):
                owned[int(table[b, p // page]), p % page] = True
        pools.append(torch.where(owned[:, None, :, None, None], pool, math.nan).to(dtype).to(device))
    return *pools, table.to(device), torch.tensor(lengths, dtype=torch.int32).to(device), refs.to(device)


def fork(k, v, table, lengths, refs, parents, page):
    """(k, v, table, lengths, refs, status) after the fork, all on the CPU."""
    k, v, table, lengths, refs = (t.cpu().clone() for t in (k, v, table, lengths, refs))
    parents = [int(p) for p in parents]
    old, was, count, pages, status = table.clone(), lengths.clone(), table.shape[0], refs.numel(), 0
    for b, p in enumerate(parents):
        if not -1 <= p < count:
            parents[b], status = b, status | 4
    keeps = {}
    for b, p in enumerate(parents):
        if p >= 0 and (p == b or p not in keeps):
            keeps[p] = b
    wants = []
    for b, p in enumerate(parents):
        if p == b:
            continue
        n = int(was[p]) if p >= 0 else 0
        full, rest = n // page, n % page
        table[b], lengths[b] = -1, n
        table[b, :full] = old[p, :full] if p >= 0 else -1
        if rest and keeps[p] == b:
            table[b, full] = old[p, full]
        elif rest:
            wants.append((b, int(old[p, full]), full, rest))
    for e in old[old >= 0].tolist():
        refs[e] -= 1
    for e in table[table >= 0].tolist():
        refs[e] += 1
    free = [i for i in range(pages) if refs[i] <= 0]
    for rank, (b, source, full, rest) in enumerate(wants):
        if rank >= len(free):
            lengths[b], status = full * page, status | 8
            continue
        table[b, full], refs[free[rank]] = free[rank], 1
        k[free[rank], :, :rest], v[free[rank], :, :rest] = k[source, :, :rest], v[source, :, :rest]
    return k, v, table, lengths, refs, status


def compact(k, v, table, refs):
    k, v, table, refs = (t.cpu().clone() for t in (k, v, table, refs))
    used = int((refs > 0).sum())
    holes = [i for i in range(used) if refs[i] <= 0]
    movers = [i for i in range(used, refs.numel()) if refs[i] > 0]
    place = list(range(refs.numel()))
    for to, source in zip(holes, movers):
        place[source] = to
        k[to], v[to] = k[source], v[source]
        refs[to], refs[source] = int(refs[source]), 0
    return k, v, torch.tensor([[place[e] if e >= 0 else e for e in row] for row in table.tolist()], dtype=torch.int32), refs, used


def select(logits, scores, finished=None, eos=None, candidates=None):
    """(scores, parents, tokens) by a sort of everything there is."""
    logits, scores = logits.cpu().to(F64), scores.cpu().to(F64)
    batch, beams, vocab = logits.shape
    count = beams if candidates is None else candidates
    out = torch.empty((batch, count), dtype=F64), torch.empty((batch, count), dtype=torch.int32), torch.empty((batch, count), dtype=torch.long)
    for b in range(batch):
        each = torch.full((beams, vocab), -math.inf, dtype=F64)
        for i in range(beams):
            if not math.isfinite(scores[b, i]):
                continue
            if finished is not None and bool(finished[b, i]):
                each[i, eos] = scores[b, i]
                continue
            lse = torch.logsumexp(logits[b, i], 0)
            if torch.isfinite(lse):
                each[i] = scores[b, i] + (logits[b, i] - lse)
        order = sorted(range(beams * vocab), key=lambda j: (-each.view(-1)[j].item(), j))[:count] if vocab < 300 else \
            torch.sort(each.view(-1), descending=True, stable=True).indices[:count].tolist()
        place = list(range(count))
        if candidates is None:
            place, left = [None] * count, [i for i in range(beams) if i not in {j // vocab for j in order}]
            met = set()
            for rank, j in enumerate(order):
                i = j // vocab
                place[rank] = left.pop(0) if i in met else i
                met.add(i)
        for rank, j in enumerate(order):
            out[0][b, place[rank]], out[1][b, place[rank]], out[2][b, place[rank]] = each.view(-1)[j], b * beams + j // vocab, j % vocab
    return out
