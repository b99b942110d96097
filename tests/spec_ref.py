"""Plain 64-bit forms of the speculative-step operators and the inputs their tests share."""
import math
import random

import numpy as np
import torch


def tree_masks(counts, rnd, kind="tree"):
    """Ancestor words (python ints, unsigned) of every drafted token."""
    out = []
    for t in counts:
        got = []
        for i in range(t):
            if kind == "tree":
                parent = rnd.randint(max(-1, i - 5), i - 1) if i else -1
            elif kind == "star":
                parent = 0 if i else -1
            else:
                parent = i - 1
            got.append((got[parent] if parent >= 0 else 0) | 1 << i)
        out += got
    return out


def mask_tensor(words, device="cuda"):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device=device)


class Paged:
    """A batch of sequences in a page pool whose unused rows hold NaN."""

    def __init__(self, seed, lens, counts, *, nkh, hd, page, spare=2, device="cuda", dtype=torch.float16):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.counts, self.nkh, self.hd, self.page = list(lens), list(counts), nkh, hd, page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).int()
        self.table_host = torch.zeros((len(lens), max(max(need, default=1), 1)), dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table_host[b, :n] = order[at:at + n]
            at += n
        self.rows = []  # (k, v) [len, nkh, hd] of each sequence
        kp = torch.full((pages, page, nkh, hd), float("nan"), dtype=dtype)
        vp = kp.clone()
        for b, n in enumerate(lens):
            k = torch.randn((n, nkh, hd), generator=g).to(dtype)
            v = torch.randn((n, nkh, hd), generator=g).to(dtype)
            self.rows.append((k, v))
            s = torch.arange(n)
            p = self.table_host[b].long()[s // page]
            kp[p, s % page] = k
            vp[p, s % page] = v
        self.k, self.v, self.table = kp.to(device), vp.to(device), self.table_host.to(device)
        self.lens_dev = torch.tensor(lens, dtype=torch.int32, device=device)
        self.indptr_host = [0] + np.cumsum(counts).tolist()
        self.indptr = torch.tensor(self.indptr_host, dtype=torch.int32, device=device)


def seen_rows(base, token, words, window):
    """Row indices (of the sequence) that drafted token `token` attends to; words None: a chain."""
    mine = list(range(token + 1)) if words is None else [j for j in range(64) if words[token] >> j & 1]
    rows = list(range(base)) + [base + j for j in mine]
    return rows[-window:] if window else rows


def tree_attn_ref(case, q, words, *, scale, window):
    """([tokens, nqh, hd] f64, largest sum |q||k| scale log2 e of a row) from the definition."""
    q = q.cpu().double()
    nqh, hd = q.shape[1], q.shape[2]
    group = nqh // case.nkh
    out = torch.zeros_like(q)
    amp = 0.0
    for b, n in enumerate(case.lens):
        t = case.counts[b]
        i0 = case.indptr_host[b]
        k, v = (x.double() for x in case.rows[b])
        mine = None if words is None else [w & ((1 << t) - 1) for w in words[i0:i0 + t]]
        for i in range(t):
            rows = seen_rows(n - t, i, mine, window)
            if not rows:
                continue
            r = torch.tensor(rows)
            for h in range(nqh):
                kk, vv = k[r, h // group], v[r, h // group]
                s = kk @ q[i0 + i, h] * scale
                amp = max(amp, float((kk.abs() @ q[i0 + i, h].abs()).max()) * abs(scale) * math.log2(math.e))
                out[i0 + i, h] = torch.softmax(s, 0) @ vv
    return out, amp


def tree_tolerance(amp, hd, keys, vmax, f16):
    """Bound of the absolute error of one output.

    A score (in powers of two) is off by amp * 2^-22 for the split of q and amp * (hd / 16 + 2) *
    2^-23 for the f32 sums of hd / 16 tensor-core steps (which truncate: one step each); a weight by
    ln 2 times that and 2^-21 for exp2 and its argument; the weighted mean by twice its weights'
    relative error (numerator and denominator) and keys / 16 + 4 more truncated sums, but never more
    than the error of adding all in sequence.  With f16 queries each weight is rounded once more
    (2^-11) and so is the output."""
    ds = amp * (2.0 ** -22 + (hd / 16 + 2) * 2.0 ** -23)
    dp = math.log(2) * ds + 2.0 ** -21
    rel = 2 * dp + (keys / 16 + 4) * 2.0 ** -23
    if f16:
        rel += 2 * 2.0 ** -11
    return rel * vmax


def prep_ref(q, k, v, qw, kw, cos_sin, nqh, nkh, hd, eps):
    """Normed and rotated q, k and normed v in f64 ([tokens, heads, hd])."""
    h = hd // 2
    cos, sin = cos_sin[:, None, :h].double(), cos_sin[:, None, h:].double()

    def norm(x, w):
        x = x.double().reshape(x.shape[0], -1, hd)
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        return y if w is None else y * w.double()

    def rot(x):
        a, b = x[..., :h], x[..., h:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    return (rot(norm(q, qw)) if nqh else None, rot(norm(k, kw)) if k is not None else None,
            norm(v, None) if v is not None else None)


def logprob_ref(x, tokens, top_k, cap):
    """(logprob, entropy, top values, top ids) in f64 from the definition."""
    raw = x.double()
    y = torch.where(raw == -math.inf, raw, cap * torch.tanh(raw / cap)) if cap else raw
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    z = e.sum(1, keepdim=True)
    lse = m + z.log()
    lp = torch.where(tokens < 0, 0.0, y.gather(1, tokens.clamp_min(0).long()) - lse)
    p = e / z
    ent = lse[:, 0] - torch.where(p > 0, p * y, 0.0).sum(1)
    key = torch.nan_to_num(raw, nan=-math.inf, posinf=math.inf, neginf=-1e300)  # NaN below -inf
    ids = key.sort(dim=1, descending=True, stable=True)[1][:, :top_k]
    return lp, ent, y.gather(1, ids) - lse, ids
