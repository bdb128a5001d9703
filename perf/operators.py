"""Cases of the text decoder's operators: paged attention of one new token, the
cache's append, fork and compact, and token log probabilities.

listed() and draw() give cases, prepare() their inputs, run() one pass: the
operators' plain form in elementary torch operations, or with `own` set the
framework's kernels. exact() gives the results of the definitions in 64 bits.

Cache tensors are (layers, pages, page, heads, head_dim) in logical order;
layout "head" stores a page head by head. Page tables are (sequences, width)
int32 with -1 past a sequence's last page.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_ops = None


def _framework():
    """The framework's public operators (wxb200.ops)."""
    global _ops
    if _ops is None:
        path = str(Path(__file__).resolve().parents[1] / "whisper-xdna_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from wxb200 import ops
        _ops = ops
    return _ops


def listed():
    return [
        # one decoder step of five beams early in a clip: the smallest call, latency counts
        {"name": "attend_beams_early", "op": "attend", "dtype": "bf16", "seqs": 5, "heads": 6,
         "group": 1, "beams": 1, "hd": 64, "page": 16, "shortest": 0, "longest": 61,
         "layout": "token", "window": False},
        # cross attention: five beams of each of 16 clips over the clip's 1500 encoder frames
        {"name": "attend_frames_1500", "op": "attend", "dtype": "bf16", "seqs": 16, "heads": 20,
         "group": 5, "beams": 5, "hd": 64, "page": 64, "shortest": 1500, "longest": 1500,
         "layout": "token", "window": False},
        # a serving batch of mixed lengths, four query heads to a key-value head
        {"name": "attend_mixed_16k", "op": "attend", "dtype": "bf16", "seqs": 64, "heads": 8,
         "group": 4, "beams": 1, "hd": 128, "page": 32, "shortest": 1, "longest": 16384,
         "layout": "token", "window": False},
        # one long sequence in fp32, few heads: the split over the cache's length carries it
        {"name": "attend_one_long_fp32", "op": "attend", "dtype": "fp32", "seqs": 1, "heads": 2,
         "group": 8, "beams": 1, "hd": 128, "page": 16, "shortest": 65519, "longest": 65519,
         "layout": "head", "window": True},
        # the keys and values of one step's new token, 64 clips of five beams
        {"name": "append_step", "op": "append", "dtype": "bf16", "seqs": 320, "heads": 20,
         "hd": 64, "page": 16, "tokens": 1, "longest": 224, "layout": "token"},
        # the encoder frames of a batch written once for cross attention
        {"name": "append_frames", "op": "append", "dtype": "bf16", "seqs": 64, "heads": 20,
         "hd": 64, "page": 64, "tokens": 1500, "longest": 1500, "layout": "token"},
        # five beams of one clip reordered after a step
        {"name": "fork_one_clip", "op": "fork", "dtype": "bf16", "clips": 1, "beams": 5,
         "done": 0, "heads": 6, "hd": 64, "page": 16, "layers": 4, "longest": 77, "spare": 16,
         "grow": 1, "layout": "token"},
        # 64 clips of five beams reordered, four of them at their end
        {"name": "fork_64_clips", "op": "fork", "dtype": "bf16", "clips": 64, "beams": 5,
         "done": 4, "heads": 20, "hd": 64, "page": 16, "layers": 8, "longest": 224, "spare": 400,
         "grow": 1, "layout": "token"},
        # a small cache made dense again
        {"name": "compact_small", "op": "compact", "dtype": "bf16", "seqs": 5, "heads": 6,
         "hd": 64, "page": 16, "layers": 4, "width": 14, "pages": 96, "moved": 11,
         "layout": "token"},
        # a server's cache made dense after many sequences ended
        {"name": "compact_server", "op": "compact", "dtype": "bf16", "seqs": 128, "heads": 8,
         "hd": 128, "page": 32, "layers": 4, "width": 32, "pages": 4001, "moved": 700,
         "layout": "head"},
        # candidates of a beam step: five rows, twice the beam's width of alternatives
        {"name": "score_beam_step", "op": "score", "dtype": "fp32", "rows": 5, "vocab": 50001,
         "top": 10, "temperature": 1.0, "masked": 90},
        # scores of whole transcripts with alternatives
        {"name": "score_transcripts", "op": "score", "dtype": "bf16", "rows": 2048,
         "vocab": 100003, "top": 5, "temperature": 0.7, "masked": 0},
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "fork", "compact", "score"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    size = 2 if dtype == "bf16" else 4
    hd = rng.choice([64, 128])
    page = rng.choice([8, 16, 32, 64, rng.randint(1, 64)])
    layout = rng.choice(["token", "head"])
    if op == "attend":
        heads, group = _log(rng, 1, 20), _log(rng, 1, 16)
        seqs = _log(rng, 1, 320)
        budget = 500e6 / (2 * heads * hd * size * seqs)
        longest = _log(rng, 1, int(max(1, min(65536, budget))))
        return {"op": op, "dtype": dtype, "seqs": seqs, "heads": heads, "group": group,
                "beams": rng.choice([1, group]), "hd": hd, "page": page,
                "shortest": rng.randint(0, longest), "longest": longest, "layout": layout,
                "window": rng.random() < 0.25}
    if op == "append":
        heads, seqs = _log(rng, 1, 20), _log(rng, 1, 320)
        tokens = _log(rng, 1, int(max(1, min(1500, 250e6 / (2 * heads * hd * size * seqs)))))
        return {"op": op, "dtype": dtype, "seqs": seqs, "heads": heads, "hd": hd, "page": page,
                "tokens": tokens, "longest": tokens + rng.randint(0, 200), "layout": layout}
    if op == "fork":
        clips, beams, heads = _log(rng, 1, 64), rng.randint(1, 8), _log(rng, 1, 20)
        grow = _log(rng, 1, 8)
        spare = clips * beams * (2 + grow // page)
        held = clips * (224 + beams * page) + spare * page      # tokens of a layer, about
        layers = max(1, min(rng.randint(1, 8), int(1.2e9 / (2 * held * heads * hd * size))))
        return {"op": op, "dtype": dtype, "clips": clips, "beams": beams,
                "done": rng.randint(0, clips // 8), "heads": heads, "hd": hd, "page": page,
                "layers": layers, "longest": _log(rng, 8, 224), "spare": spare, "grow": grow,
                "layout": layout}
    if op == "compact":
        seqs, width = _log(rng, 4, 128), _log(rng, 4, 32)
        used = seqs * (width - width // 4) + width // 4
        moved = rng.randint(1, used // 2)
        return {"op": op, "dtype": dtype, "seqs": seqs, "heads": _log(rng, 1, 8), "hd": hd,
                "page": min(page, 32), "layers": rng.randint(1, 2), "width": width,
                "pages": used + moved + rng.randint(0, used // 2), "moved": moved,
                "layout": layout}
    vocab = _log(rng, 1000, 131072)
    rows = _log(rng, 1, int(min(4096, 400e6 / (vocab * size))))
    return {"op": "score", "dtype": dtype, "rows": rows, "vocab": vocab,
            "top": rng.randint(0, 20), "temperature": rng.choice([1.0, 0.6, 1.3]),
            "masked": rng.choice([0, 90])}


# ------------------------------------------------------------------ inputs


def _lengths(n, lo, hi):
    """n lengths spread over [lo, hi] in the logarithm of length + 1: the same
    ones for every seed (the seed deals them out)."""
    if n == 1:
        return [hi]
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * i / (n - 1)) - 1)) for i in range(n)]


def _pages(n, page):
    return (n + page - 1) // page


def _noise(gen, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device=gen.device)
    return out.normal_(generator=gen)


def _pool(gen, layers, pages, case):
    """A cache of `pages` pages: (layers, pages, page, heads, hd)."""
    page, heads, hd = case["page"], case["heads"], case["hd"]
    dtype = DTYPES[case["dtype"]]
    if case["layout"] == "head":
        return _noise(gen, (layers, pages, heads, page, hd), dtype).transpose(2, 3)
    return _noise(gen, (layers, pages, page, heads, hd), dtype)


def _table(lens, page, width, ids):
    """Page table of sequences that share nothing, their pages dealt from ids."""
    table = torch.full((len(lens), max(1, width)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        k = _pages(n, page)
        table[i, :k] = ids[at:at + k]
        at += k
    return table


def _beam_lens(case):
    """Lengths before a fork, one for each clip."""
    clips, longest = case["clips"], case["longest"]
    return [max(1, n) for n in _lengths(clips, longest // 3, longest)]


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    state = {"case": case}
    if op == "score":
        # logits of a trained model: a broad bulk with a few strong candidates
        x = _noise(gen, (case["rows"], case["vocab"]), torch.float32).mul_(2.5)
        hot = torch.randint(0, case["vocab"], (case["rows"], 8), generator=gen, device=dev)
        x.scatter_add_(1, hot, _noise(gen, hot.shape, torch.float32).mul_(2).add_(9))
        if case["masked"]:
            # suppressed tokens, as a decoder masks them
            off = torch.randperm(case["vocab"], generator=host)[:case["masked"]]
            x[:, off.to(dev)] = -math.inf
        state["logits"] = x.to(dtype)
        state["tokens"] = hot[:, 0].contiguous()
        return state
    page = case["page"]
    if op in ("attend", "append"):
        lens = _lengths(case["seqs"], case.get("shortest", case.get("tokens")), case["longest"])
        lens = [lens[i] for i in torch.randperm(len(lens), generator=host).tolist()]
        used = sum(_pages(n, page) for n in lens)
        ids = torch.randperm(used + 3, generator=host).to(torch.int32)
        width = _pages(case["longest"], page)
        state["table"] = _table(lens, page, width, ids).to(dev)
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        state["k"] = _pool(gen, 1, used + 3, case)[0]
        state["v"] = _pool(gen, 1, used + 3, case)[0]
        if op == "append":
            shape = (case["seqs"], case["tokens"], case["heads"], case["hd"])
            state["k_new"], state["v_new"] = _noise(gen, shape, dtype), _noise(gen, shape, dtype)
            return state
        group, heads, hd = case["group"], case["heads"], case["hd"]
        if case["beams"] > 1:
            # the beams of a clip attend to the same keys: one group of queries
            q = _noise(gen, (case["seqs"] * group, heads * hd), dtype)
            state["q"] = q.view(case["seqs"], group, heads, hd).transpose(1, 2)
        else:
            q = _noise(gen, (case["seqs"], heads * group * hd), dtype)
            state["q"] = q.view(case["seqs"], heads, group, hd)
        state["starts"] = None
        if case["window"]:
            # the cache's first tokens are outside the window
            starts = [_start(n) for n in lens]
            state["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        return state
    if op == "fork":
        beams, lens = case["beams"], _beam_lens(case)
        full = [n // page for n in lens]
        need = sum(f + beams * (_pages(n, page) - f) for f, n in zip(full, lens))
        pages = need + case["spare"]
        width = _pages(case["longest"] + case["grow"], page)
        ids = torch.randperm(pages, generator=host).to(torch.int32)
        table = torch.full((len(lens) * beams, width), -1, dtype=torch.int32)
        at = 0
        for c, n in enumerate(lens):
            rows = table[c * beams:(c + 1) * beams]
            rows[:, :full[c]] = ids[at:at + full[c]]   # whole pages are shared by the beams
            at += full[c]
            if n % page:
                rows[:, full[c]] = ids[at:at + beams]  # each beam writes in a page of its own
                at += beams
        parents = []
        for c in range(len(lens)):
            turn = torch.randperm(beams, generator=host)
            parents.append(c * beams + turn[torch.arange(beams) // 2])
        parents = torch.stack(parents).to(torch.int32)
        parents[len(lens) - case["done"]:] = -1        # these clips are at their end
        state["parents"] = parents.reshape(-1).to(dev)
        grow = torch.full((len(lens), beams), case["grow"], dtype=torch.int32)
        grow[len(lens) - case["done"]:] = 0
        state["grow"] = grow.reshape(-1).to(dev)
        state["lens"] = torch.tensor(lens, dtype=torch.int32).repeat_interleave(beams).to(dev)
    else:
        seqs, width = case["seqs"], case["width"]
        shared = width // 4
        n_used = shared + seqs * (width - shared)
        low = torch.randperm(n_used, generator=host)[:n_used - case["moved"]]
        high = n_used + torch.randperm(case["pages"] - n_used, generator=host)[:case["moved"]]
        ids = torch.cat([low, high])[torch.randperm(n_used, generator=host)].to(torch.int32)
        table = torch.empty(seqs, width, dtype=torch.int32)
        table[:, :shared] = ids[:shared]               # a prefix that all sequences share
        table[:, shared:] = ids[shared:].view(seqs, width - shared)
        pages = case["pages"]
    held = table[table >= 0].long()
    state["refs"] = torch.bincount(held, minlength=pages).to(torch.int32).to(dev)
    state["table"] = table.to(dev)
    state["k"] = _pool(gen, case["layers"], pages, case)
    state["v"] = _pool(gen, case["layers"], pages, case)
    return state


def _start(n):
    return n // 3


# ------------------------------------------------------------------ plain forms


def _attend(q, k, v, table, lens, starts):
    S, H, G, hd = q.shape
    at = table.long().clamp(min=0)
    keys = k[at].reshape(S, -1, H, hd).float().permute(0, 2, 1, 3)
    values = v[at].reshape(S, -1, H, hd).float().permute(0, 2, 1, 3)
    pos = torch.arange(keys.shape[2], device=q.device)
    seen = pos < lens[:, None]
    if starts is not None:
        seen &= pos >= starts[:, None]
    s = torch.matmul(q.float(), keys.transpose(2, 3)) * (1 / math.sqrt(hd))
    s = torch.where(seen[:, None, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    values = torch.where(seen[:, None, :, None], values, 0.0)
    o = torch.matmul(e, values) / torch.where(total == 0, 1.0, total)
    lse = (m + torch.log(total))[..., 0]
    return {"o": o.to(q.dtype), "lse": lse}


def _append(k_new, v_new, k, v, table, lens):
    S, T = k_new.shape[:2]
    page = k.shape[1]
    pos = (lens[:, None] - T + torch.arange(T, device=k.device)).long()
    at = torch.gather(table.long(), 1, pos // page)
    k[at, pos % page] = k_new
    v[at, pos % page] = v_new
    return {"k": k, "v": v}


def _fork(k, v, table, lens, refs, parents, grow):
    S, width = table.shape
    pages, page = refs.shape[0], k.shape[2]
    dev = table.device
    ids = torch.arange(S, device=dev)
    cols = torch.arange(width, device=dev)
    alive = parents >= 0
    par = parents.long().clamp(min=0)
    now = torch.where(alive, lens[par], 0).long()
    held = (now + page - 1) // page
    rows = torch.where(alive[:, None] & (cols < held[:, None]), table[par].long(), -1)
    # references: the old rows' are given back, the new rows' are taken
    count = refs.long().clone()
    for_rows = lambda r, sign: count.index_add_(  # noqa: E731
        0, r.clamp(min=0).reshape(-1), torch.where(r >= 0, sign, 0).reshape(-1))
    for_rows(table.long(), -1)
    for_rows(rows, 1)
    # a partly filled page that others refer to is copied, but for its keeper: the
    # longest of them, the first among equals
    part = now % page
    last = torch.gather(rows, 1, (now // page).clamp(max=width - 1)[:, None])[:, 0]
    wants = (grow > 0) & (now + grow <= width * page)
    other = rows[:, (now // page).clamp(max=width - 1)].T      # row i: every row's page there
    mate = (other == last[:, None]) & (last >= 0)[:, None]
    rank = now * S + (S - 1 - ids)
    best = torch.where(mate, rank, -1).amax(1) == rank
    copies = wants & (part > 0) & (count[last.clamp(min=0)] > 1) & ~best
    fresh = torch.where(wants, (now + grow + page - 1) // page - held, 0)
    need = copies.long() + fresh
    before = need.cumsum(0) - need
    free = count == 0
    n_free = free.sum()
    granted = wants & ((need == 0) | (before + need <= n_free))
    order = torch.sort(torch.where(free, 0, 1), stable=True).indices  # free pages, ascending
    take = lambda n: order[n.clamp(max=pages - 1)]  # noqa: E731
    copies &= granted
    src = last.clamp(min=0)
    dst = take(before)
    first = before + copies.long()
    new = granted[:, None] & (cols >= held[:, None]) & (cols < (held + fresh)[:, None])
    rows = torch.where(new, take(first[:, None] + cols - held[:, None]), rows)
    rows = torch.where(copies[:, None] & (cols == (now // page)[:, None]), dst[:, None], rows)
    count.index_add_(0, src, torch.where(copies, -1, 0))
    count.index_add_(0, rows.clamp(min=0).reshape(-1), new.long().reshape(-1))
    count.index_add_(0, dst, copies.long())
    # the copied tokens, all layers at once
    s, d, n = src[copies], dst[copies], part[copies]
    kept = (torch.arange(page, device=dev) < n[:, None])[None, :, :, None, None]
    k[:, d] = torch.where(kept, k[:, s], k[:, d])
    v[:, d] = torch.where(kept, v[:, s], v[:, d])
    grown = torch.where(granted, grow, 0)
    total = need.sum()
    left = (count == 0).sum()
    status = torch.stack([left, (total - n_free).clamp(min=0)]).to(torch.int32)
    return {"table": rows.to(torch.int32), "lens": (now + grown).to(torch.int32),
            "refs": count.to(torch.int32), "grown": grown.to(torch.int32), "status": status,
            "k": k, "v": v}


def _compact(k, v, table, refs):
    pages = refs.shape[0]
    ids = torch.arange(pages, device=refs.device)
    used = refs > 0
    n_used = used.sum()
    holes = ids[~used & (ids < n_used)]
    movers = ids[used & (ids >= n_used)]
    to = ids.clone()
    to[movers] = holes
    k[:, holes] = k[:, movers]
    v[:, holes] = v[:, movers]
    table = torch.where(table >= 0, to[table.long().clamp(min=0)].to(torch.int32), -1)
    refs = torch.where(ids < n_used, refs.index_select(0, _inverse(to, movers, holes)), 0)
    return {"table": table, "refs": refs, "k": k, "v": v,
            "status": torch.stack([n_used, torch.as_tensor(movers.numel(), device=refs.device)])
            .to(torch.int32)}


def _inverse(to, movers, holes):
    back = torch.arange(to.shape[0], device=to.device)
    back[holes] = movers
    return back


def _score(logits, tokens, top, temperature):
    z = logits.float() / temperature
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    logprob = torch.gather(z, 1, tokens[:, None])[:, 0] - lse[:, 0]
    mean = torch.where(e > 0, e * d, 0.0).sum(1) / total[:, 0]
    out = {"logprob": logprob, "entropy": torch.log(total)[:, 0] - mean}
    index = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
    out["top_logprob"] = torch.gather(z, 1, index) - lse
    out["top_index"] = index.to(torch.int32)
    return out


# ------------------------------------------------------------------ one pass


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        if op == "attend":
            return _attend(state["q"], state["k"], state["v"], state["table"], state["lens"],
                           state["starts"])
        if op == "append":
            return _append(state["k_new"], state["v_new"], state["k"], state["v"],
                           state["table"], state["lens"])
        if op == "fork":
            return _fork(state["k"], state["v"], state["table"], state["lens"], state["refs"],
                         state["parents"], state["grow"])
        if op == "compact":
            return _compact(state["k"], state["v"], state["table"], state["refs"])
        return _score(state["logits"], state["tokens"], case["top"], case["temperature"])
    ops = _framework()
    if op == "attend":
        o, lse = ops.paged_attention(state["q"], state["k"], state["v"], state["table"],
                                     state["lens"], starts=state["starts"], return_lse=True)
        return {"o": o, "lse": lse}
    if op == "append":
        ops.kv_append(state["k_new"], state["v_new"], state["k"], state["v"], state["table"],
                      state["lens"])
        return {"k": state["k"], "v": state["v"]}
    if op == "fork":
        table, lens, refs, grown, status = ops.kv_fork(
            state["k"], state["v"], state["table"], state["lens"], state["refs"],
            parents=state["parents"], grow=state["grow"])
        return {"table": table, "lens": lens, "refs": refs, "grown": grown, "status": status,
                "k": state["k"], "v": state["v"]}
    if op == "compact":
        table, refs, status = ops.kv_compact(state["k"], state["v"], state["table"],
                                             state["refs"])
        return {"table": table, "refs": refs, "k": state["k"], "v": state["v"],
                "status": status}
    logprob, entropy, top_logprob, top_index = ops.token_logprobs(
        state["logits"], state["tokens"], top_k=case["top"], temperature=case["temperature"])
    return {"logprob": logprob, "entropy": entropy, "top_logprob": top_logprob,
            "top_index": top_index}


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    """The floating results by definition in float64 (copies of cache pages and whole
    numbers have none)."""
    if case["op"] == "attend":
        s = prepare(case, seed)
        q, page = s["q"].double(), case["page"]
        S, H, G, hd = q.shape
        o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
        for i, n in enumerate(s["lens"].tolist()):
            first = 0 if s["starts"] is None else int(s["starts"][i])
            if first >= n:
                continue
            pos = torch.arange(first, n, device=q.device)
            at = s["table"][i].long()[torch.div(pos, page, rounding_mode="floor")]
            for h in range(H):
                x = q[i, h] @ s["k"][at, pos % page, h].double().T / math.sqrt(hd)
                lse[i, h] = torch.logsumexp(x, 1)
                p = torch.exp(x - lse[i, h][:, None])
                o[i, h] = p @ s["v"][at, pos % page, h].double()
        return {"o": o, "lse": lse}
    if case["op"] == "score":
        s = prepare(case, seed)
        out = {"logprob": [], "entropy": [], "top_logprob": []}
        for r in range(0, case["rows"], 256):
            x = s["logits"][r:r + 256].double() / case["temperature"]
            lp = x - torch.logsumexp(x, 1, keepdim=True)
            out["logprob"].append(lp.gather(1, s["tokens"][r:r + 256, None])[:, 0])
            out["entropy"].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(1))
            out["top_logprob"].append(lp.topk(case["top"], dim=1).values)
        return {k: torch.cat(v) for k, v in out.items()} | {"top_index": None}
    return None


# ------------------------------------------------------------------ work


def work(case):
    op = case["op"]
    size = 2 if case["dtype"] == "bf16" else 4
    if op == "score":
        n = case["rows"] * case["vocab"]
        # one exponential, one sum and one product for each logit
        return {"bytes": n * size + case["rows"] * (8 + 8 + 8 * case["top"]), "flops": 4 * n}
    row = case["heads"] * case["hd"] * size
    if op == "attend":
        lens = _lengths(case["seqs"], case["shortest"], case["longest"])
        kept = sum(n - (_start(n) if case["window"] else 0) for n in lens)
        rows = case["seqs"] * case["heads"] * case["group"]
        held = sum(_pages(n, case["page"]) for n in lens)
        return {"bytes": 2 * kept * row + rows * (2 * case["hd"] * size + 4) + 4 * held,
                "flops": 4 * kept * case["heads"] * case["group"] * case["hd"]}
    if op == "append":
        return {"bytes": 4 * case["seqs"] * case["tokens"] * row + 8 * case["seqs"], "flops": 0}
    if op == "fork":
        # a clip's beams but its parents copy the part of a page that is filled
        page, beams = case["page"], case["beams"]
        live = _beam_lens(case)
        copied = sum((n % page) * (beams // 2) for n in live[:len(live) - case["done"]])
        width = _pages(case["longest"] + case["grow"], page)
        tables = 2 * 4 * case["clips"] * beams * width
        return {"bytes": 2 * 2 * case["layers"] * copied * row + tables, "flops": 0}
    moved = 2 * 2 * case["layers"] * case["moved"] * case["page"] * row
    return {"bytes": moved + 8 * case["seqs"] * case["width"] + 8 * case["pages"], "flops": 0}
