"""The operators of a long-context step over the paged cache: what they compute, on which sizes they are timed.

A serving program whose prompts are longer than one pass and whose caches are kept to a budget:

  chunk   attention of a chunk of new tokens of every sequence (a piece of a prompt, or one decoded token) over the
          paged cache: causal, or a sliding window beside a few first tokens that stay visible
  mass    the attention weight that every cached row has got from the chunk's tokens, added to what it had
  evict   the rows with the most accumulated weight kept, with the first and the latest ones, and moved together

`run` computes each in a plain form of elementary torch operations, or (own = True) through g4attn.Context.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoded token of one sequence in a sliding layer with four sinks: the smallest call, where latency counts
        {"name": "chunk_one", "op": "chunk", "batch": 1, "tokens": 1, "length": 4000, "ragged": False, "nqh": 8, "nkh": 1,
         "hd": 256, "page": 64, "window": 512, "sinks": 4},
        # one decoded token of each of 64 sequences over all of their rows: the cache has to be read once
        {"name": "chunk_decode", "op": "chunk", "batch": 64, "tokens": 1, "length": 12000, "ragged": True, "nqh": 8,
         "nkh": 1, "hd": 256, "page": 64, "window": 0, "sinks": 0},
        # a piece of a prompt in a sliding layer
        {"name": "chunk_sliding", "op": "chunk", "batch": 1, "tokens": 2048, "length": 6000, "ragged": False, "nqh": 8,
         "nkh": 1, "hd": 256, "page": 64, "window": 512, "sinks": 4},
        # a piece of a prompt in a global layer (head_dim 512), an odd number of tokens
        {"name": "chunk_global", "op": "chunk", "batch": 1, "tokens": 1001, "length": 20003, "ragged": False, "nqh": 8,
         "nkh": 1, "hd": 512, "page": 64, "window": 0, "sinks": 0},
        # unequal pieces of six prompts, three q heads for each of four kv heads, small pages
        {"name": "chunk_ragged", "op": "chunk", "batch": 6, "tokens": 700, "length": 9000, "ragged": True, "nqh": 12,
         "nkh": 4, "hd": 128, "page": 16, "window": 0, "sinks": 0},
        # the end of a long document: 512 tokens over 131,000 rows
        {"name": "chunk_long", "op": "chunk", "batch": 1, "tokens": 512, "length": 131000, "ragged": False, "nqh": 8,
         "nkh": 1, "hd": 256, "page": 64, "window": 0, "sinks": 0},
        # one decoded token's weights over a cache at its budget: latency
        {"name": "mass_one", "op": "mass", "batch": 1, "tokens": 1, "length": 4000, "ragged": False, "nqh": 8, "nkh": 1,
         "hd": 256, "page": 64, "window": 0, "sinks": 0, "decay": 1.0},
        # a decode step of 24 sequences in a global layer, older weight fading
        {"name": "mass_decode", "op": "mass", "batch": 24, "tokens": 1, "length": 16000, "ragged": True, "nqh": 8, "nkh": 1,
         "hd": 512, "page": 64, "window": 0, "sinks": 0, "decay": 0.98},
        # a piece of a prompt: all of its tokens look back over 32,000 rows
        {"name": "mass_chunk", "op": "mass", "batch": 1, "tokens": 515, "length": 32000, "ragged": False, "nqh": 8, "nkh": 1,
         "hd": 256, "page": 16, "window": 0, "sinks": 0, "decay": 1.0},
        # one sequence back to its budget
        {"name": "evict_one", "op": "evict", "batch": 1, "length": 4096, "budget": 2048, "sinks": 4, "recent": 256,
         "ragged": False, "nkh": 1, "hd": 256, "page": 64},
        # a long prompt cut to an eighth
        {"name": "evict_long", "op": "evict", "batch": 1, "length": 131000, "budget": 16384, "sinks": 4, "recent": 512,
         "ragged": False, "nkh": 1, "hd": 512, "page": 64},
        # a batch of prompts of unequal length, every one of four kv heads with rows of its own
        {"name": "evict_batch", "op": "evict", "batch": 24, "length": 9000, "budget": 4097, "sinks": 4, "recent": 300,
         "ragged": True, "nkh": 4, "hd": 128, "page": 16},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    hi = max(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "mass", "mass", "evict"])
    nkh = rng.choice([1, 1, 2, 4])
    page = rng.choice([8, 16, 16, 48, 64, 64, 128])
    hd = rng.choice([64, 96, 128, 256, 256, 512])
    if op == "evict":
        batch = _spread(rng, 1, 32)
        length = _spread(rng, 2, min(131000, 131000 * 512 // (batch * nkh * hd)))
        budget = _spread(rng, 1, length)
        sinks = rng.choice([0, min(4, budget)])
        return {"op": op, "batch": batch, "length": length, "budget": budget, "sinks": sinks,
                "recent": rng.randint(0, (budget - sinks) // 2), "ragged": rng.random() < 0.7, "nkh": nkh, "hd": hd,
                "page": page}
    nqh = nkh * rng.choice([1, 3, 4, 8, 8])
    batch = _spread(rng, 1, 64)
    # the scores of the plain form stay within those of the largest listed case of the operator
    most = (512 * 8 * 131000 if op == "chunk" else 515 * 8 * 32000) // (batch * nqh)
    tokens = 1 if rng.random() < 0.3 else _spread(rng, 1, min(2048, math.isqrt(most)))
    length = _spread(rng, tokens, min(131000, most // tokens, 131000 * 512 // (batch * nkh * hd)))
    c = {"op": op, "batch": batch, "tokens": min(tokens, length), "length": length, "ragged": rng.random() < 0.7, "nqh": nqh,
         "nkh": nkh, "hd": hd, "page": page, "window": rng.choice([0, 0, 512, _spread(rng, 1, 2000)])}
    c["sinks"] = rng.choice([0, 4, _spread(rng, 1, 200)]) if c["window"] else 0
    if op == "mass":
        c["decay"] = rng.choice([1.0, 1.0, 0.98, 0.0])
    return c


# ------------------------------------------------------------------------------------- sizes of one case

def _tokens_of(c):
    top, r = c["tokens"], random.Random(17)
    return [r.randint(1 + top // 3, top) if c["ragged"] and b else top for b in range(c["batch"])]


def _lens_of(c):
    """Rows of each sequence in the cache, the new tokens' own among them."""
    r = random.Random(29)
    low = c["length"] // 3
    new = [1] * c["batch"] if c["op"] == "evict" else _tokens_of(c)
    return [max(t, r.randint(low, c["length"]) if c["ragged"] and b else c["length"]) for b, t in enumerate(new)]


def _seen(c, n, t):
    """Rows that the last t of n tokens read, and the pairs (token, row) that are seen."""
    w, s = c["window"], c["sinks"]
    if not w or w >= n:
        return n, t * n - t * (t - 1) // 2
    first = max(0, n - t + 1 - w)
    pairs = sum(min(p, w) + min(s, max(0, p - w)) for p in range(n - t + 1, n + 1))
    return n - first + min(s, first), pairs


def work(c):
    row = c["nkh"] * c["hd"] * 2
    if c["op"] == "evict":
        kept = sum(min(n, c["budget"]) - c["sinks"] for n in _lens_of(c) if n > c["budget"])
        read = sum(n for n in _lens_of(c) if n > c["budget"])
        return {"bytes": kept * row * 4 + read * c["nkh"] * 4 + kept * c["nkh"] * 8, "flops": 0}
    keys = pairs = 0
    for t, n in zip(_tokens_of(c), _lens_of(c)):
        k, p = _seen(c, n, t)
        keys, pairs = keys + k, pairs + p
    rows = sum(_tokens_of(c)) * c["nqh"]
    if c["op"] == "chunk":
        return {"bytes": 2 * keys * row + rows * (4 * c["hd"] + 4), "flops": 4 * pairs * c["nqh"] * c["hd"]}
    old = sum(_lens_of(c)) - sum(_tokens_of(c)) if c["decay"] else 0
    return {"bytes": keys * row + rows * (2 * c["hd"] + 4) + 4 * c["nkh"] * (old + sum(_lens_of(c))),
            "flops": 2 * pairs * c["nqh"] * c["hd"]}


# ---------------------------------------------------------------------------------------------- inputs

def _pages(lens, page, gen, spare=3):
    """A page table whose pages lie in a random order, as in a pool that has been in use."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen, device=DEV).int()
    table = torch.zeros((len(lens), max(max(need), 1)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    randn = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    lens = _lens_of(c)
    s = {"case": c, "lens": ints(lens), "longest": max(lens)}
    s["table"], pages = _pages(lens, c["page"], gen)
    s["k_pages"], s["v_pages"] = (
        torch.randn((pages, c["page"], c["nkh"], c["hd"]), generator=gen, device=DEV, dtype=torch.float16) for _ in range(2))
    if c["op"] == "evict":
        # accumulated weights: a few rows with much, most with little, some that no token has looked at
        mass = (randn(c["batch"], c["nkh"], s["longest"]) * 2).exp()
        s["mass"] = mass * (torch.rand(mass.shape, generator=gen, device=DEV) > 0.1)
        s["new_lens"] = torch.zeros_like(s["lens"])
        s["kept"] = torch.zeros((c["batch"], c["nkh"], c["budget"]), dtype=torch.int32, device=DEV)
        return s
    new = _tokens_of(c)
    s["most"] = max(new)
    s["indptr"] = ints([sum(new[:b]) for b in range(len(new) + 1)])
    # normed queries whose scores spread over a few units, as a trained q norm leaves them
    s["q"] = (randn(sum(new), c["nqh"], c["hd"]) * 3).half()
    s["lse"] = torch.zeros((sum(new), c["nqh"]), device=DEV)
    if c["op"] == "chunk":
        s["out"] = torch.zeros_like(s["q"])
    else:
        # what the attention of the same tokens has left, and what the rows have got from earlier tokens
        score = _scores(s)
        s["lse"].copy_(_to_tokens(s, score.logsumexp(-1)))
        s["mass"] = randn(c["batch"], c["nkh"], s["longest"]).exp()
    return s


# ---------------------------------------------------------------------------------- the framework's calls

_context = None


def _ctx():
    global _context
    if _context is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma4-webgpu_b200"))
        import g4attn
        _context = g4attn.Context(0)
    return _context


def _run_own(s):
    c, ctx = s["case"], _ctx()
    if c["op"] == "chunk":
        ctx.chunk_attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["indptr"], s["out"], s["lse"],
                             num_q_heads=c["nqh"], num_kv_heads=c["nkh"], head_dim=c["hd"], page_size=c["page"],
                             scale=c["hd"] ** -0.5, sliding_window=c["window"], sink_tokens=c["sinks"])
        return {"out": s["out"], "lse": s["lse"]}
    if c["op"] == "mass":
        ctx.paged_key_mass(s["q"], s["lse"], s["k_pages"], s["table"], s["lens"], s["indptr"], s["mass"],
                           num_q_heads=c["nqh"], num_kv_heads=c["nkh"], head_dim=c["hd"], page_size=c["page"],
                           scale=c["hd"] ** -0.5, sliding_window=c["window"], sink_tokens=c["sinks"], decay=c["decay"])
        return s["mass"]
    ctx.paged_kv_evict(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["mass"], s["new_lens"], s["kept"],
                       budget=c["budget"], sink_tokens=c["sinks"], recent_tokens=c["recent"], num_kv_heads=c["nkh"],
                       head_dim=c["hd"], page_size=c["page"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "mass": s["mass"], "new_lens": s["new_lens"],
            "kept": s["kept"]}


# -------------------------------------------------------------------------------------- the plain forms

def _rows_of(s):
    """Rows of q of a padded batch [batch, most], and which of them are there."""
    first = s["indptr"].long()
    t = torch.arange(s["most"], device=DEV)
    live = t < (first[1:] - first[:-1])[:, None]
    return torch.where(live, first[:-1, None] + t, 0), live


def _cached(s, pool):
    """Cache rows of a padded batch in 32 bits, [batch, keys, nkh, hd]."""
    c = s["case"]
    key = torch.arange(s["longest"], device=DEV)
    at = s["table"][:, key // c["page"]].long() * c["page"] + key % c["page"]
    return pool.view(-1, c["nkh"], c["hd"])[at].float()


def _scores(s):
    """Scaled scores [batch, nkh, most, group, keys] in 32 bits, -inf where a token does not see a row."""
    c = s["case"]
    rows, live = _rows_of(s)
    group = c["nqh"] // c["nkh"]
    q = s["q"][rows].float().view(*rows.shape, c["nkh"], group, c["hd"]).permute(0, 2, 1, 3, 4)
    score = q.reshape(c["batch"], c["nkh"], -1, c["hd"]) @ _cached(s, s["k_pages"]).permute(0, 2, 3, 1)
    score = score.view(c["batch"], c["nkh"], s["most"], group, s["longest"]).mul_(c["hd"] ** -0.5)
    key = torch.arange(s["longest"], device=DEV)
    # a token's own row: the last ones of its sequence are the new tokens'
    own_row = (s["lens"] - s["indptr"].diff())[:, None, None] + torch.arange(s["most"], device=DEV)[:, None]
    seen = (key <= own_row) & live[..., None]
    if c["window"]:
        seen = seen & ((key > own_row - c["window"]) | (key < c["sinks"]))
    return score.masked_fill_(~seen[:, None, :, None], -math.inf)


def _to_tokens(s, x):
    """[batch, nkh, most, group, ...] of the padded batch to the tokens' rows [tokens, nqh, ...]."""
    _, live = _rows_of(s)
    x = x.transpose(1, 2)
    return x.reshape(*x.shape[:2], s["case"]["nqh"], *x.shape[4:])[live]


def _plain_chunk(s):
    c = s["case"]
    score = _scores(s)
    top = score.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    e = score.sub_(top).exp_()
    z = e.sum(-1, keepdim=True)
    out = e.view(c["batch"], c["nkh"], -1, s["longest"]) @ _cached(s, s["v_pages"]).transpose(1, 2)
    out = out.view(*z.shape[:-1], c["hd"]) / z.masked_fill(z == 0, 1.0)
    s["out"].copy_(_to_tokens(s, out))
    s["lse"].copy_(_to_tokens(s, (z.log() + top)[..., 0]))
    return {"out": s["out"], "lse": s["lse"]}


def _plain_mass(s):
    c = s["case"]
    score = _scores(s)
    rows, _ = _rows_of(s)
    lse = s["lse"][rows].view(*rows.shape, c["nkh"], -1).permute(0, 2, 1, 3)
    got = score.sub_(lse[..., None]).exp_().sum((2, 3))
    key = torch.arange(s["longest"], device=DEV)
    old = (key < (s["lens"] - s["indptr"].diff())[:, None])[:, None]
    there = (key < s["lens"][:, None])[:, None]
    kept = torch.where(old, s["mass"] * c["decay"], 0.0) if c["decay"] else 0.0
    s["mass"].copy_(torch.where(there, kept + got, s["mass"]))
    return s["mass"]


def _plain_evict(s):
    c = s["case"]
    budget, lens = c["budget"], s["lens"].long()
    key = torch.arange(s["longest"], device=DEV)
    n = lens[:, None, None]
    # order of the rows: those that stay in any case, then by weight, the earlier one first among equals
    sure = (key < c["sinks"]) | (key >= n - c["recent"])
    rank = (s["mass"].view(torch.int32).long() + 1).masked_fill(sure, 1 << 31).masked_fill(key >= n, 0)
    rank = (rank << 24) + (s["longest"] - 1 - key)
    kept = (s["longest"] - 1 - (rank.topk(min(budget, s["longest"]), -1)[0] & 0xffffff)).sort(-1)[0]
    slot = torch.arange(kept.shape[-1], device=DEV)
    kept = torch.where(n <= budget, slot.expand_as(kept), kept)
    there = (slot < n).expand_as(kept)
    s["kept"].fill_(-1)
    s["kept"][..., :kept.shape[-1]] = torch.where(there, kept, -1)
    s["new_lens"].copy_(lens.clamp(max=budget))
    moved = there & (n > budget)
    s["mass"][..., :kept.shape[-1]] = torch.where(moved, s["mass"].gather(-1, kept), s["mass"][..., :kept.shape[-1]])
    b, h, i = moved.nonzero(as_tuple=True)
    j = kept[moved]
    src = s["table"][b, j // c["page"]].long() * c["page"] + j % c["page"]
    dst = s["table"][b, i // c["page"]].long() * c["page"] + i % c["page"]
    for pool in (s["k_pages"], s["v_pages"]):
        rows = pool.view(-1, c["nkh"], c["hd"])
        rows[dst, h] = rows[src, h]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "mass": s["mass"], "new_lens": s["new_lens"],
            "kept": s["kept"]}


def run(state):
    if own:
        return _run_own(state)
    return {"chunk": _plain_chunk, "mass": _plain_mass, "evict": _plain_evict}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------- the definitions, 64 bits

def _sequence(s, b, pool):
    """The cache rows of one sequence, [rows, nkh, hd] in 64 bits."""
    c, n = s["case"], int(s["lens"][b])
    i = torch.arange(n, device=DEV)
    return pool.view(-1, c["nkh"], c["hd"])[s["table"][b].long()[i // c["page"]] * c["page"] + i % c["page"]].double()


def _weights(s, b, k):
    """Pieces of a sequence's tokens: (slice of q's rows, scores [tokens, nkh, group, rows]) in 64 bits."""
    c, first, n = s["case"], s["indptr"].tolist(), len(k)
    t = first[b + 1] - first[b]
    step = max(1, 200_000_000 // (n * c["nqh"]))
    row = torch.arange(n, device=DEV)
    for t0 in range(0, t, step):
        part = slice(first[b] + t0, first[b] + min(t, t0 + step))
        q = s["q"][part].double().view(part.stop - part.start, c["nkh"], -1, c["hd"])
        x = torch.einsum("tkgd,nkd->tkgn", q, k) / math.sqrt(c["hd"])
        last = n - t + t0 + torch.arange(len(q), device=DEV)[:, None]
        hidden = row > last
        if c["window"]:
            hidden |= (row <= last - c["window"]) & (row >= c["sinks"])
        yield part, x.masked_fill_(hidden[:, None, None], -math.inf)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "chunk":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=DEV)
        for b in range(c["batch"]):
            k, v = _sequence(s, b, s["k_pages"]), _sequence(s, b, s["v_pages"])
            for part, x in _weights(s, b, k):
                lse[part] = torch.logsumexp(x, -1).flatten(1)
                out[part] = torch.einsum("tkgn,nkd->tkgd", torch.softmax(x, -1), v).flatten(1, 2)
        return {"out": out, "lse": lse}
    if c["op"] == "mass":
        mass, first = s["mass"].double(), s["indptr"].tolist()
        for b in range(c["batch"]):
            k = _sequence(s, b, s["k_pages"])
            n, t = len(k), first[b + 1] - first[b]
            total = torch.zeros((c["nkh"], n), dtype=torch.float64, device=DEV)
            total[:, :n - t] = mass[b, :, :n - t] * c["decay"]
            for part, x in _weights(s, b, k):
                lse = s["lse"][part].double().view(*x.shape[:3], 1)
                total += torch.exp(x - lse).sum((0, 2))
            mass[b, :, :n] = total
        return mass
    k, v, mass = s["k_pages"].clone(), s["v_pages"].clone(), s["mass"].clone()
    kept = torch.full_like(s["kept"], -1)
    page, first, recent, budget = c["page"], c["sinks"], c["recent"], c["budget"]
    for b, n in enumerate(s["lens"].tolist()):
        if n <= budget:
            kept[b, :, :n] = torch.arange(n, device=DEV)
            continue
        for h in range(c["nkh"]):
            middle = s["mass"][b, h, first:n - recent].sort(descending=True, stable=True)[1][:budget - first - recent] + first
            stay = torch.cat([torch.arange(first, device=DEV), middle.sort()[0], torch.arange(n - recent, n, device=DEV)])
            kept[b, h] = stay
            mass[b, h, :budget] = s["mass"][b, h, stay]
            place = lambda i: (s["table"][b].long()[i // page], i % page)  # noqa: E731
            (p, r), (x, y) = place(torch.arange(budget, device=DEV)), place(stay)
            k[p, r, h], v[p, r, h] = s["k_pages"][x, y, h], s["v_pages"][x, y, h]
    return {"k_pages": k, "v_pages": v, "mass": mass, "new_lens": s["lens"].clamp(max=budget), "kept": kept}
