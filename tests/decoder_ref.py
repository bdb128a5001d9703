"""Plain restatements of the decoder operators for the tests: attention and
scores from their definitions in 64 bits with bounds on what fp32 and bf16
arithmetic may be off, and the cache's page plans written out step by step in
Python."""
import math

import torch

U32 = 2.0 ** -24     # unit roundoff of fp32
U16 = 2.0 ** -9      # half of bf16's


def attend64(q, k_cache, v_cache, table, lens, scale, starts=None):
    """(o, lse, o's bound, lse's bound) in float64. q (S, H, G, hd).

    Bounds, with a_j = scale sum |q||k_j| and A = max_j a_j: a score carries at
    most (hd + 3) u A; a weight twice that, the exponential's 2^-22 and the
    exponent's rounding (|s_j - m| <= 2 A, in log2 units: 2 A 2^-23); a sum of n
    terms n u. A bf16 result is rounded once, 2^-8 |o|, which is at most 2^-9
    sum p|v| + 2^-9 |o|; its weights have to be kept to more bits than bf16's."""
    q, dev = q.double(), q.device
    S, H, G, hd = q.shape
    page = k_cache.shape[1]
    bf16 = k_cache.dtype == torch.bfloat16
    o = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=dev)
    o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    for i, n in enumerate(lens.tolist()):
        first = 0 if starts is None else max(0, int(starts[i]))
        if first >= n:
            continue
        pos = torch.arange(first, n, device=dev)
        at = table[i].long()[pos // page]
        k = k_cache[at, pos % page].double()      # (n, H, hd)
        v = v_cache[at, pos % page].double()
        s = torch.einsum("hgd,nhd->hgn", q[i], k) * scale
        A = (torch.einsum("hgd,nhd->hgn", q[i].abs(), k.abs()) * abs(scale)).amax(-1)
        lse[i] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[i][..., None])
        o[i] = torch.einsum("hgn,nhd->hgd", p, v)
        spread = torch.einsum("hgn,nhd->hgd", p, v.abs())
        m = n - first
        w = 2 * (hd + 3) * U32 * A + 2.0 ** -22 + 2 * A * 2.0 ** -23 + (m + 64) * U32
        lse_tol[i] = w + lse[i].abs() * 2.0 ** -22
        off = (2 * w)[..., None] * spread
        if bf16:
            off = off + U16 * spread
            off = off + U16 * (o[i].abs() + off)
        o_tol[i] = off + 1e-30
    return o, lse, o_tol, lse_tol


def score64(logits, tokens, top_k, temperature):
    """(logprob, entropy, top_logprob, top_index, their bounds) in float64.

    With d = z - max z: an exponent carries |d| 2^-22, an exponential 2^-22, a
    sum over the row at most (vocab / 256 + 64) u (the longest chain of one
    thread and the tree above it)."""
    x = logits.double()
    z = x / temperature
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = m + torch.log(total)
    ad = torch.where(e > 0, d.abs(), 0.0)
    n = (x.shape[1] / 256 + 64) * U32
    rel = (p * (ad * 2.0 ** -22)).sum(1) + 2.0 ** -22 + n      # of the sum
    inside = (tokens >= 0) & (tokens < x.shape[1])
    zt = z.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp = torch.where(inside, zt - lse[:, 0], torch.where(tokens < 0, 0.0, -math.inf))
    mean = (p * ad).sum(1)
    ent = torch.log(total)[:, 0] + mean
    step = lambda t: t.abs() * 2.0 ** -22 + 1e-7  # noqa: E731
    # each term of the mean carries its weight's error times its depth
    mean_off = (p * ad * (ad * 2.0 ** -22 + 2.0 ** -21)).sum(1) + mean * (rel + n)
    index = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top_k]
    top = z.gather(1, index) - lse
    return {"logprob": lp, "entropy": ent, "top_logprob": top, "top_index": index,
            "logprob_tol": rel + step(zt - m[:, 0]) + step(lp.clamp(min=-1e30)),
            "entropy_tol": rel + mean_off + step(ent) + 1e-6,
            "top_tol": rel[:, None] + step(top.clamp(min=-1e30)) + step(
                (z.gather(1, index) - m).clamp(min=-1e30))}


def fork_ref(table, lens, refs, parents, grow, page):
    """One fork on Python lists. Returns (table, lens, refs, grown, status, copies)
    with copies a list of (source page, target page, tokens)."""
    S, width = len(table), len(table[0])
    pages = lambda n: (n + page - 1) // page  # noqa: E731
    parents = list(range(S)) if parents is None else parents
    grow = [0] * S if grow is None else grow
    now = [lens[p] if p >= 0 else 0 for p in parents]
    rows = [table[p][:pages(n)] if p >= 0 else [] for p, n in zip(parents, now)]
    rows = [list(r) for r in rows]
    refs = list(refs)
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] -= 1
    for row in rows:
        for p in row:
            refs[p] += 1
    free = [p for p, r in enumerate(refs) if r == 0]
    n_free, asked = len(free), 0
    shared = {}
    for i, row in enumerate(rows):
        if row and now[i] % page:
            users = [j for j in range(S) if row[-1] in rows[j]]
            keeper = max(users, key=lambda j: (now[j], -j))
            shared[i] = len(users) > 1 and keeper != i
    grown, copies, out = [0] * S, [], [list(r) for r in rows]
    for i in range(S):
        g = max(0, grow[i])
        if g == 0 or now[i] + g > width * page:
            continue
        copy = shared.get(i, False)
        need = pages(now[i] + g) - pages(now[i]) + copy
        take = free[asked:asked + need]
        asked += need
        if need and asked > n_free:
            continue
        grown[i] = g
        if copy:
            src, dst = rows[i][-1], take.pop(0)
            copies.append((src, dst, now[i] % page))
            out[i][-1] = dst
            refs[src] -= 1
            refs[dst] += 1
        for p in take:
            out[i].append(p)
            refs[p] += 1
    table = [r + [-1] * (width - len(r)) for r in out]
    status = [sum(r == 0 for r in refs), max(0, asked - n_free)]
    return table, [n + g for n, g in zip(now, grown)], refs, grown, status, copies


def compact_ref(table, refs):
    """One compaction on Python lists: (table, refs, status, moves)."""
    used = [p for p, r in enumerate(refs) if r > 0]
    n = len(used)
    holes = [p for p in range(n) if refs[p] == 0]
    movers = [p for p in used if p >= n]
    to = {m: h for m, h in zip(movers, holes)}
    new = [refs[p] if p < n else 0 for p in range(len(refs))]
    for m, h in to.items():
        new[h] = refs[m]
    return ([[to.get(p, p) for p in row] for row in table], new, [n, len(movers)],
            list(to.items()))
