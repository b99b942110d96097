"""Plain 64-bit forms of the long-context operators and the error bounds of their kernels."""
import math

import torch


def seen(n, t, window, sinks, device="cuda"):
    """[t, n] truth values: which of n rows the last t tokens see."""
    row = torch.arange(n, device=device)
    pos = n - t + torch.arange(t, device=device)[:, None]
    s = row <= pos
    if window:
        s &= (row > pos - window) | (row < sinks)
    return s


def chunk_ref(case, q, *, scale, window=0, sinks=0, there=None):
    """out [tokens, nqh, hd], lse [tokens, nqh] in f64, and amp, the largest sum |q||k| scale log2 e of a pair.  there
    ([rows] truth values of each sequence) leaves rows out."""
    q = q.double()
    nqh, hd = q.shape[1], q.shape[2]
    group = nqh // case.nkh
    out, lse, amp = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device), 0.0
    for b, n in enumerate(case.lens):
        t, i0 = case.counts[b], case.indptr_host[b]
        if t == 0:
            continue
        k, v = (x.cuda().double() for x in case.rows[b])
        s = seen(n, t, window, sinks)
        if there is not None:
            s = s & there[b].cuda()
        for h in range(nqh):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[i0:i0 + t, h]
            amp = max(amp, float((qq.abs() @ kk.abs().T).max()) * abs(scale) * math.log2(math.e))
            x = (qq @ kk.T * scale).masked_fill(~s, -math.inf)
            z = torch.logsumexp(x, 1)
            lse[i0:i0 + t, h] = z
            w = torch.exp(x - z.masked_fill(z == -math.inf, 0.0)[:, None])
            out[i0:i0 + t, h] = w @ vv
    return out, lse, amp


def mass_ref(case, q, lse, mass, *, scale, window=0, sinks=0, decay=1.0):
    """mass after the call, [batch, nkh, stride] in f64."""
    q, lse, got = q.double(), lse.double(), mass.double()
    group = q.shape[1] // case.nkh
    for b, n in enumerate(case.lens):
        t, i0 = case.counts[b], case.indptr_host[b]
        got[b, :, :n - t] = got[b, :, :n - t] * decay if decay else 0.0
        got[b, :, n - t:n] = 0.0
        if t == 0:
            continue
        k = case.rows[b][0].cuda().double()
        s = seen(n, t, window, sinks)
        for h in range(q.shape[1]):
            z = lse[i0:i0 + t, h, None]
            w = torch.exp(q[i0:i0 + t, h] @ k[:, h // group].T * scale - z)
            got[b, h // group, :n] += torch.where(s & (z > -math.inf), w, 0.0).sum(0)
    return got


def score_error(amp, hd):
    """Of a score in powers of two: the f32 sums of hd / 16 tensor-core steps (which truncate: one step each) and the
    products with the scale and its log2 e."""
    return amp * (hd / 16 + 4) * 2.0 ** -23


def attn_tolerance(amp, hd, keys, vmax):
    """Bound of the absolute error of one f16 output: a weight is off by ln 2 times the score's error and 2^-21 for exp2
    and its argument, twice (numerator and denominator), and by its rounding to f16, 2^-11 relative or 2^-25 (the
    largest weight is 2^-1 at least, so that is 2^-24 of their sum for each key); keys / 16 + 36 additions of f32; the output's rounding."""
    dp = math.log(2) * score_error(amp, hd) + 2.0 ** -21
    return (2 * dp + 2.0 ** -11 + keys * 2.0 ** -24 + (keys / 16 + 36) * 2.0 ** -23 + 2.0 ** -11) * vmax


def lse_tolerance(amp, hd, keys, top):
    """Of a log-sum-exp: the score's error, the sum's relative error, and three roundings at its size (top)."""
    return math.log(2) * score_error(amp, hd) + 2.0 ** -21 + (keys / 16 + 36) * 2.0 ** -24 + 3 * top * 2.0 ** -24


def mass_tolerance(amp, hd, rows, top):
    """Relative, of one entry: a weight as above with lse's size (top) rounded twice in powers of two, and `rows` + 2
    additions (in the worst order)."""
    return math.log(2) * (score_error(amp, hd) + 2 * (top * math.log2(math.e) + 1) * 2.0 ** -24) + 2.0 ** -21 + \
        (rows + 2) * 2.0 ** -24


def evict_ref(mass, lens, *, budget, sinks, recent):
    """kept [batch, nkh, budget] (python lists, -1 behind) of masses on the CPU."""
    out = []
    for b, n in enumerate(lens):
        heads = []
        for h in range(mass.shape[1]):
            if n <= budget:
                heads.append(list(range(n)) + [-1] * (budget - n))
                continue
            m = mass[b, h].tolist()
            key = lambda r: (-math.inf if m[r] != m[r] else m[r], 0 if m[r] != m[r] else 1)  # noqa: E731
            middle = sorted(range(sinks, n - recent), key=lambda r: (key(r), -r), reverse=True)
            heads.append(sorted(list(range(sinks)) + middle[:budget - sinks - recent] + list(range(n - recent, n))))
        out.append(heads)
    return torch.tensor(out, dtype=torch.int32)
