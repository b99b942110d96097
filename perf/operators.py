"""The operators of a speculative step over the paged cache: what they compute, on which sizes they are timed.

A step of a serving program that lets a draft model propose a tree of tokens for every sequence:

  prep      norms and rotation of the new tokens' q and k heads, v norm, and the append of k and v to the paged cache
  tree      attention of the drafted tokens over the cache, each seeing the prefix and its own ancestors
  logprob   log probabilities of the proposed tokens under the target's logits, entropy and top alternatives
  compact   the accepted path's rows moved to the places that the next step expects them in

`run` computes each in a plain form of elementary torch operations, or (own = True) through g4attn.Context.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoded token of one sequence in a sliding layer: the smallest append, where latency counts
        {"name": "prep_one", "op": "prep", "batch": 1, "per_seq": 1, "ragged": False, "far": 4000, "nqh": 8, "nkh": 1,
         "hd": 256, "page": 64, "fmt": "f32", "fused": False, "consumer": False},
        # 16 sequences' trees in a global layer, q / k / v as columns of one projection's output
        {"name": "prep_trees", "op": "prep", "batch": 16, "per_seq": 24, "ragged": True, "far": 30000, "nqh": 8,
         "nkh": 1, "hd": 512, "page": 64, "fmt": "f32", "fused": True, "consumer": False},
        # prompt chunks of five sequences, an odd number of tokens, q kept in 16 bits for the tensor cores
        {"name": "prep_chunks", "op": "prep", "batch": 5, "per_seq": 1801, "ragged": True, "far": 8000, "nqh": 8,
         "nkh": 1, "hd": 256, "page": 16, "fmt": "f16", "fused": False, "consumer": False},
        # one sequence, eight drafted tokens, a sliding layer of 512 keys: latency
        {"name": "tree_sliding", "op": "tree", "batch": 1, "tokens": 8, "length": 2000, "ragged": False, "nqh": 8,
         "nkh": 1, "hd": 256, "page": 64, "window": 512, "tree": True, "fmt": "f32"},
        # eight sequences of unequal length with trees of up to 24 tokens, all keys, 32-bit queries
        {"name": "tree_batch", "op": "tree", "batch": 8, "tokens": 24, "length": 12000, "ragged": True, "nqh": 8,
         "nkh": 1, "hd": 256, "page": 64, "window": 0, "tree": True, "fmt": "f32"},
        # one long context in a global layer (head_dim 512), a tree of 48 tokens, 16-bit queries
        {"name": "tree_long", "op": "tree", "batch": 1, "tokens": 48, "length": 131000, "ragged": False, "nqh": 8,
         "nkh": 1, "hd": 512, "page": 64, "window": 0, "tree": True, "fmt": "f16"},
        # many short sequences, three q heads for each of four kv heads, small pages, chains of drafted tokens
        {"name": "tree_chains", "op": "tree", "batch": 32, "tokens": 7, "length": 3000, "ragged": True, "nqh": 12,
         "nkh": 4, "hd": 128, "page": 16, "window": 0, "tree": False, "fmt": "f16"},
        # the next token of one sequence over the whole vocabulary, capped logits, 20 alternatives
        {"name": "logprob_one", "op": "logprob", "rows": 1, "vocab": 262144, "tokens": 1, "top": 20, "cap": 30.0,
         "fmt": "f32"},
        # 37 rows of a smaller odd vocabulary in 16 bits, four children each, greedy choice and runners-up
        {"name": "logprob_odd", "op": "logprob", "rows": 37, "vocab": 50257, "tokens": 4, "top": 5, "cap": 0.0,
         "fmt": "f16"},
        # the trees of a whole batch: 384 rows over the vocabulary
        {"name": "logprob_batch", "op": "logprob", "rows": 384, "vocab": 262144, "tokens": 3, "top": 8, "cap": 30.0,
         "fmt": "f32"},
        # one sequence's accepted path of four tokens: latency
        {"name": "compact_one", "op": "compact", "batch": 1, "accept": 4, "length": 1000, "nkh": 1, "hd": 256,
         "page": 64},
        # 64 sequences, up to 16 tokens each, global layer rows
        {"name": "compact_batch", "op": "compact", "batch": 64, "accept": 16, "length": 900, "nkh": 1, "hd": 512,
         "page": 16},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prep", "tree", "tree", "logprob", "compact"])
    nkh = rng.choice([1, 1, 2, 4])
    heads = {"nqh": nkh * rng.choice([1, 3, 4, 8, 8]), "nkh": nkh}
    page = rng.choice([8, 16, 16, 48, 64, 64, 128])
    fmt = rng.choice(["f32", "f16"])
    if op == "prep":
        hd, batch = rng.choice([64, 128, 256, 256, 512]), _spread(rng, 1, 32)
        per_seq = _spread(rng, 1, max(1, min(1800, 40_000_000 // (batch * hd * (heads["nqh"] + 2 * nkh)))))
        return {"op": op, "batch": batch, "per_seq": per_seq, "ragged": rng.random() < 0.7, "far": _spread(rng, 16, 30000),
                **heads, "hd": hd, "page": page, "fmt": fmt, "fused": rng.random() < 0.5, "consumer": rng.random() < 0.15}
    if op == "tree":
        hd = rng.choice([64, 96, 128, 256, 256, 512])
        batch, tokens = _spread(rng, 1, 32), _spread(rng, 1, 64)
        # the scores of the plain form stay within those of the largest listed case
        most = 48 * 8 * 131000 // (batch * tokens * heads["nqh"])
        most = min(most, 131000 * 512 // (batch * nkh * hd), 131000)
        return {"op": op, "batch": batch, "tokens": tokens, "length": _spread(rng, tokens, max(tokens, most)),
                "ragged": rng.random() < 0.7, **heads, "hd": hd, "page": page,
                "window": rng.choice([0, 0, 512, _spread(rng, 1, 2000)]), "tree": rng.random() < 0.7, "fmt": fmt}
    if op == "logprob":
        vocab = rng.choice([262144, 262144, 32000, 50257, _spread(rng, 100, 200000)])
        return {"op": op, "rows": _spread(rng, 1, 384 * 262144 // vocab if vocab > 40000 else 1500), "vocab": vocab,
                "tokens": rng.choice([1, 1, 2, 4, 7]), "top": rng.choice([0, 1, 5, 8, 20, 32]),
                "cap": rng.choice([0.0, 30.0]), "fmt": fmt}
    return {"op": op, "batch": _spread(rng, 1, 64), "accept": _spread(rng, 1, 32), "length": _spread(rng, 1, 900),
            "nkh": nkh, "hd": rng.choice([64, 128, 256, 512]), "page": page}


# ------------------------------------------------------------------------------------- sizes of one case

def _tokens_of(c):
    """New tokens of each sequence (prep: prompt chunk or tree; tree: drafted tokens)."""
    top, r = c["per_seq"] if c["op"] == "prep" else c["tokens"], random.Random(17)
    return [r.randint(1 + top // 3, top) if c["ragged"] and b else top for b in range(c["batch"])]


def _lens_of(c):
    """Rows of each sequence in the cache, the drafted ones among them (tree)."""
    r = random.Random(29)
    return [max(t, r.randint(c["length"] // 3, c["length"]) if c["ragged"] and b else c["length"])
            for b, t in enumerate(_tokens_of(c))]


def _starts_of(c):
    """Rows that each sequence has in the cache before the call (prep, compact)."""
    r, top = random.Random(23), c["far"] if c["op"] == "prep" else c["length"]
    return [r.randint(top // 2, top) for _ in range(c["batch"])]


def _accepts_of(c):
    r = random.Random(31)
    return [r.randint(0, c["accept"]) if b else c["accept"] for b in range(c["batch"])]


def work(c):
    size = 4 if c.get("fmt") == "f32" else 2
    if c["op"] == "prep":
        n, kv = sum(_tokens_of(c)), 0 if c["consumer"] else 2 * c["nkh"]
        heads = c["nqh"] + kv
        return {"bytes": n * c["hd"] * (4 * heads + 4 + size * c["nqh"] + 2 * kv), "flops": n * c["hd"] * 8 * heads}
    if c["op"] == "tree":
        keys = seen = 0
        for t, n in zip(_tokens_of(c), _lens_of(c)):
            keys += min(n, c["window"] + t) if c["window"] else n
            seen += t * (min(n, c["window"]) if c["window"] else n - t // 2)
        return {"bytes": keys * c["nkh"] * c["hd"] * 4 + sum(_tokens_of(c)) * c["nqh"] * c["hd"] * 2 * size,
                "flops": 4 * seen * c["nqh"] * c["hd"]}
    if c["op"] == "logprob":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * (8 * c["tokens"] + 4 + 8 * c["top"]), "flops": 8 * n}
    return {"bytes": sum(_accepts_of(c)) * c["nkh"] * c["hd"] * 2 * 4 + 16 * c["batch"], "flops": 0}


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


def _pool(pages, c, gen):
    return [torch.randn((pages, c["page"], c["nkh"], c["hd"]), generator=gen, device=DEV, dtype=torch.float16)
            for _ in range(2)]


def _tree_masks(counts, tree, rnd):
    """Ancestor bits of each drafted token (its own among them): parents drawn among the earlier tokens."""
    masks = []
    for t in counts:
        got = []
        for i in range(t):
            parent = -1 if i == 0 else rnd.randint(max(-1, i - 6), i - 1) if tree else i - 1
            m = (got[parent] if parent >= 0 else 0) | (1 << i)
            got.append(m)
        masks += got
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    rnd = random.Random(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    randn = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    s = {"case": c}
    if c["op"] == "prep":
        new = _tokens_of(c)
        n, hd, nqh, nkh = sum(new), c["hd"], c["nqh"], c["nkh"]
        start = _starts_of(c)
        s["table"], pages = _pages([a + t for a, t in zip(start, new)], c["page"], gen)
        s["k_pages"], s["v_pages"] = _pool(pages, c, gen)
        where = [a + i for a, t in zip(start, new) for i in range(t)]
        s["slots"] = ints(where)
        s["token_seq"] = ints([b for b, t in enumerate(new) for _ in range(t)])
        # cos and sin of the tokens' angles, which a forward pass has once for all of its layers
        inv = 10000.0 ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float64) * 2 / hd)
        angle = torch.tensor(where, device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        if c["fused"]:
            whole = randn(n, (nqh + 2 * nkh) * hd) * 2
            s["q"], s["k"], s["v"] = whole.split([nqh * hd, nkh * hd, nkh * hd], 1)
        else:
            s["q"], s["k"], s["v"] = randn(n, nqh * hd) * 2, randn(n, nkh * hd) * 2, randn(n, nkh * hd)
        if c["consumer"]:
            s["k"] = s["v"] = None
        s["q_w"], s["k_w"] = ((1 + 0.2 * randn(hd)).half() for _ in range(2))
        s["q_out"] = torch.zeros((n, nqh, hd), device=DEV, dtype=torch.float32 if c["fmt"] == "f32" else torch.float16)
    elif c["op"] == "tree":
        new, lens = _tokens_of(c), _lens_of(c)
        s["lens"], s["host_lens"], s["max_tokens"] = ints(lens), np.array(lens, dtype=np.int32), max(new)
        s["indptr"] = ints([0] + np.cumsum(new).tolist())
        s["table"], pages = _pages(lens, c["page"], gen)
        s["k_pages"], s["v_pages"] = _pool(pages, c, gen)
        s["mask"] = torch.tensor(_tree_masks(new, True, rnd), dtype=torch.int64, device=DEV) if c["tree"] else None
        # normed queries whose scores spread over a few units, as a trained q norm leaves them
        q = randn(sum(new), c["nqh"], c["hd"]) * 3
        s["q"] = q if c["fmt"] == "f32" else q.half()
        s["out"] = torch.zeros_like(s["q"])
    elif c["op"] == "logprob":
        x = randn(c["rows"], c["vocab"]) * 3
        x.scatter_add_(1, torch.randint(c["vocab"], (c["rows"], 4), generator=gen, device=DEV), 8 + 6 * randn(c["rows"], 4).abs())
        s["logits"] = x if c["fmt"] == "f32" else x.half()
        s["tokens"] = torch.randint(c["vocab"], (c["rows"], c["tokens"]), generator=gen, device=DEV).int()
        s["tokens"][:, 0] = x.argmax(1).int()
        s["logprob"] = torch.zeros((c["rows"], c["tokens"]), device=DEV)
        s["entropy"] = torch.zeros(c["rows"], device=DEV)
        s["top"] = torch.zeros((c["rows"], c["top"]), device=DEV)
        s["top_ids"] = torch.zeros((c["rows"], c["top"]), dtype=torch.int32, device=DEV)
    else:
        base = _starts_of(c)
        s["table"], pages = _pages([b + 64 for b in base], c["page"], gen)
        s["k_pages"], s["v_pages"] = _pool(pages, c, gen)
        # an accepted path through a tree of 64 nodes: a stem that stays where it is, then scattered nodes
        path = np.full((c["batch"], c["accept"]), -1, dtype=np.int32)
        for b, n in enumerate(_accepts_of(c)):
            stem = rnd.randint(0, n // 2)
            path[b, :n] = list(range(stem)) + sorted(rnd.sample(range(n, 64), n - stem))
        s["base"], s["path"], s["path_lens"] = ints(base), torch.from_numpy(path).to(DEV), ints(_accepts_of(c))
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
    if c["op"] == "prep":
        ctx.paged_qkv_prep(s["q"], s["k"], s["v"], s["q_w"], s["k_w"], s["cos_sin"], s["q_out"], s["k_pages"],
                           s["v_pages"], s["table"], s["token_seq"], s["slots"], num_q_heads=c["nqh"],
                           num_kv_heads=c["nkh"], head_dim=c["hd"], page_size=c["page"], eps=1e-6)
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if c["op"] == "tree":
        ctx.tree_attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["indptr"], s["mask"], s["out"],
                            num_q_heads=c["nqh"], num_kv_heads=c["nkh"], head_dim=c["hd"], page_size=c["page"],
                            max_tokens=s["max_tokens"], scale=c["hd"] ** -0.5, sliding_window=c["window"],
                            host_kv_lens=s["host_lens"])
        return s["out"]
    if c["op"] == "logprob":
        ctx.token_logprobs(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["top"], s["top_ids"],
                           softcap=c["cap"])
        return {"logprob": s["logprob"], "entropy": s["entropy"], "top": s["top"], "top_ids": s["top_ids"]}
    ctx.paged_kv_compact(s["k_pages"], s["v_pages"], s["table"], s["base"], s["path"], s["path_lens"],
                         num_kv_heads=c["nkh"], head_dim=c["hd"], page_size=c["page"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# -------------------------------------------------------------------------------------- the plain forms

def _plain_prep(s):
    c = s["case"]
    n, hd, half = s["q"].shape[0], c["hd"], c["hd"] // 2
    cos, sin = s["cos_sin"][:, None, :half], s["cos_sin"][:, None, half:]

    def normed(x, w):
        x = x.reshape(n, -1, hd)
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        return y if w is None else y * w.float()

    def rotated(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    s["q_out"].copy_(rotated(normed(s["q"], s["q_w"])))
    if s["k"] is not None:
        slot, seq = s["slots"].long(), s["token_seq"].long()
        row = s["table"][seq, slot // c["page"]].long() * c["page"] + slot % c["page"]
        s["k_pages"].view(-1, c["nkh"], hd)[row] = rotated(normed(s["k"], s["k_w"])).half()
        s["v_pages"].view(-1, c["nkh"], hd)[row] = normed(s["v"], None).half()
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_tree(s):
    c = s["case"]
    nkh, hd, group = c["nkh"], c["hd"], c["nqh"] // c["nkh"]
    lens, first = s["lens"].long(), s["indptr"].long()
    count = first[1:] - first[:-1]
    most, longest, batch = s["max_tokens"], int(s["host_lens"].max()), len(lens)
    t = torch.arange(most, device=DEV)
    live = t < count[:, None]
    row = torch.where(live, first[:-1, None] + t, first[:-1, None])  # [batch, most]
    # which drafted tokens each token sees, and how many come before each of them
    bit = torch.arange(64, device=DEV)
    if s["mask"] is None:
        sees = (bit <= t[:, None]).expand(batch, most, 64)
    else:
        sees = (s["mask"][row][..., None] >> bit & 1) == 1
    sees = sees & live[..., None]
    total, rank = sees.sum(-1), sees.cumsum(-1) - sees.long()
    base = lens - count
    key = torch.arange(longest, device=DEV)
    draft = (key - base[:, None]).clamp(0, 63)[:, None].expand(batch, most, longest)
    old = (key < base[:, None])[:, None]
    seen = (old | sees.gather(2, draft)) & (key < lens[:, None])[:, None] & live[..., None]
    if c["window"]:
        place = torch.where(old, key, base[:, None, None] + rank.gather(2, draft))
        seen = seen & (place >= (base[:, None] + total - c["window"])[..., None])
    at = s["table"][:, key // c["page"]].long() * c["page"] + key % c["page"]
    k = s["k_pages"].view(-1, nkh, hd)[at].float().permute(0, 2, 3, 1)  # [batch, nkh, hd, keys]
    v = s["v_pages"].view(-1, nkh, hd)[at].float().permute(0, 2, 1, 3)
    q = s["q"][row].float().view(batch, most, nkh, group, hd).permute(0, 2, 1, 3, 4).reshape(batch, nkh, -1, hd)
    score = (q @ k * hd ** -0.5).view(batch, nkh, most, group, longest)
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - top.masked_fill(top == -math.inf, 0.0)).exp_()
    z = e.sum(-1, keepdim=True)
    out = e.view(batch, nkh, -1, longest) @ v
    out = out.view(batch, nkh, most, group, hd) / z.masked_fill(z == 0, 1.0)
    s["out"][row[live]] = out.permute(0, 2, 1, 3, 4).reshape(batch, most, -1, hd)[live].to(s["out"].dtype)
    return s["out"]


def _plain_logprob(s):
    c = s["case"]
    raw = s["logits"].float()
    x = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
    x = x - x.amax(1, keepdim=True)
    e = x.exp()
    z = e.sum(1, keepdim=True, dtype=torch.float64)
    log_z = z.log()
    s["logprob"].copy_(x.gather(1, s["tokens"].long()) - log_z)
    s["entropy"].copy_((log_z - (e * x).sum(1, keepdim=True, dtype=torch.float64) / z)[:, 0])
    if c["top"]:
        # the largest logits, the lower id first among equal ones: keys of the value's bits, in order, above the id's
        bits = (raw + 0.0).view(torch.int32)
        bits = (bits ^ (bits >> 31 & 0x7fffffff)).long() << 32
        ids = c["vocab"] - 1 - ((bits + torch.arange(c["vocab"] - 1, -1, -1, device=DEV)).topk(c["top"], 1)[0] & 0xffffffff)
        s["top_ids"].copy_(ids)
        s["top"].copy_(x.gather(1, ids) - log_z)
    return {"logprob": s["logprob"], "entropy": s["entropy"], "top": s["top"], "top_ids": s["top_ids"]}


def _plain_compact(s):
    c = s["case"]
    i = torch.arange(s["path"].shape[1], device=DEV)
    live = i < s["path_lens"][:, None]
    b = torch.arange(len(s["base"]), device=DEV)[:, None].expand_as(live)[live]
    src = (s["base"][:, None] + s["path"])[live].long()
    dst = (s["base"][:, None] + i)[live].long()
    src = s["table"][b, src // c["page"]].long() * c["page"] + src % c["page"]
    dst = s["table"][b, dst // c["page"]].long() * c["page"] + dst % c["page"]
    k, v = (s[n].view(-1, c["nkh"], c["hd"]) for n in ("k_pages", "v_pages"))
    k[dst], v[dst] = k[src], v[src]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def run(state):
    if own:
        return _run_own(state)
    return {"prep": _plain_prep, "tree": _plain_tree, "logprob": _plain_logprob, "compact": _plain_compact}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------- the definitions, 64 bits

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "prep":
        n, hd, h = s["q"].shape[0], c["hd"], c["hd"] // 2
        w = torch.complex(s["cos_sin"][:, :h].double(), s["cos_sin"][:, h:].double())[:, None]

        def head(x, weight=None):
            x = x.double().reshape(n, -1, hd)
            y = x * ((x * x).sum(-1, keepdim=True) / hd + 1e-6) ** -0.5
            if weight is None:
                return y
            y = y * weight.double()
            z = torch.complex(y[..., :h], y[..., h:]) * w  # a pair turned by its angle
            return torch.cat([z.real, z.imag], -1)

        k, v = s["k_pages"].double(), s["v_pages"].double()
        if s["k"] is not None:
            seq, slot = s["token_seq"].tolist(), s["slots"].tolist()
            table = s["table"].tolist()
            at = torch.tensor([table[b][i // c["page"]] * c["page"] + i % c["page"] for b, i in zip(seq, slot)], device=DEV)
            k.view(-1, c["nkh"], hd)[at] = head(s["k"], s["k_w"])
            v.view(-1, c["nkh"], hd)[at] = head(s["v"])
        return {"q": head(s["q"], s["q_w"]), "k_pages": k, "v_pages": v}
    if c["op"] == "tree":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        first, lens = s["indptr"].tolist(), s["lens"].tolist()
        mask = None if s["mask"] is None else [m & (2 ** 64 - 1) for m in s["mask"].tolist()]
        group = c["nqh"] // c["nkh"]
        for b, n in enumerate(lens):
            t = first[b + 1] - first[b]
            base = n - t
            i = torch.arange(n, device=DEV)
            at = s["table"][b].long()[i // c["page"]] * c["page"] + i % c["page"]
            k = s["k_pages"].view(-1, c["nkh"], c["hd"])[at].double()
            v = s["v_pages"].view(-1, c["nkh"], c["hd"])[at].double()
            seen = torch.zeros((t, n), dtype=torch.bool, device=DEV)
            for j in range(t):
                mine = [x for x in range(t) if (x <= j if mask is None else mask[first[b] + j] >> x & 1)]
                drop = max(0, base + len(mine) - c["window"]) if c["window"] else 0
                seen[j, min(drop, base):base] = True
                kept = mine[max(0, drop - base):]
                seen[j, torch.tensor([base + x for x in kept], dtype=torch.long, device=DEV)] = True
            q = s["q"][first[b]:first[b + 1]].double().view(t, c["nkh"], group, c["hd"])
            p = torch.einsum("tkgd,nkd->tkgn", q, k) / math.sqrt(c["hd"])
            p = torch.softmax(p.masked_fill(~seen[:, None, None], -math.inf), -1)
            out[first[b]:first[b + 1]] = torch.einsum("tkgn,nkd->tkgd", p, v).reshape(t, c["nqh"], c["hd"])
        return out
    if c["op"] == "logprob":
        got = {"logprob": [], "entropy": [], "top": []}
        ids = s["logits"].sort(dim=1, descending=True, stable=True)[1][:, :c["top"]]
        for x, tok, top in zip(s["logits"], s["tokens"].long(), ids):
            x = x.double()
            x = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
            lp = torch.log_softmax(x, 0)
            got["logprob"].append(lp[tok])
            got["entropy"].append(-(lp.exp() * lp).sum())
            got["top"].append(lp[top])
        return {**{k: torch.stack(v) for k, v in got.items()}, "top_ids": ids.int()}
    k, v, page = s["k_pages"].clone(), s["v_pages"].clone(), c["page"]
    table, base = s["table"].tolist(), s["base"].tolist()
    for b, (path, n) in enumerate(zip(s["path"].tolist(), s["path_lens"].tolist())):
        for i, j in enumerate(path[:n]):
            x, y = base[b] + j, base[b] + i
            for pool, old in ((k, s["k_pages"]), (v, s["v_pages"])):
                pool[table[b][y // page], y % page] = old[table[b][x // page], x % page]
    return {"k_pages": k, "v_pages": v}
