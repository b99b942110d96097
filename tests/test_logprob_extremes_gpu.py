"""Log probabilities of rows with huge finite logits: tokens banned by a large negative value instead of -inf, the
type's lowest and largest values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
LOWEST = torch.finfo(torch.float32).min


def _reference(x, tokens, k, cap):
    """In 64 bits, the maximum taken out first: y - (m + ln S) loses ln S where m is huge."""
    raw = x.double()
    y = cap * torch.tanh(raw / cap) if cap else raw
    y = y - y.amax(1, keepdim=True)
    s = torch.exp(y).sum(1, keepdim=True)
    lp = y - s.log()
    p = torch.exp(lp)
    ids = raw.sort(dim=1, descending=True, stable=True)[1][:, :k]
    return lp.gather(1, tokens.long()), s.log()[:, 0] - (p * y).sum(1), lp.gather(1, ids), ids


def _check(ctx, x, tokens, k, cap=0.0):
    """log p = (y - m) - ln S: two roundings of 2^-24 of its parts (the difference, log p), so 2^-22 |log p| at most, and
    the error of ln S, that of S relative: exponents off by 2^-24 |d| with weights e^d, of which sum |d| e^d <= S ln V,
    exp2 2^-22, f32 sums of less than 64 terms in sequence and in trees 2^-20 - together below 2^-18 for ln V <= 13.  The
    entropy ln S - T / S has T / S <= ln V, T and S as exact as S above: 2^-18 (1 + ln V).  A capped
    logit is off by 2^-22 of the largest in its row, and so is the maximum."""
    rows, vocab = x.shape
    lp = torch.full(tokens.shape, 9.0, device="cuda")
    ent = torch.full((rows,), 9.0, device="cuda")
    tv = torch.full((rows, k), 9.0, device="cuda")
    ti = torch.full((rows, k), -9, dtype=torch.int32, device="cuda")
    ctx.token_logprobs(x, tokens, lp, ent, tv, ti, softcap=cap)
    ctx.sync()
    rlp, rent, rtv, rti = _reference(x.cpu(), tokens.cpu(), k, cap)
    assert torch.equal(ti.cpu().long(), rti)
    raw = x.cpu().double()
    size = (cap * torch.tanh(raw / cap)).abs().amax(1, keepdim=True) if cap else torch.zeros((rows, 1))
    tol = 2.0 ** -18 + size * 2.0 ** -21
    for got, want in ((lp, rlp), (tv, rtv)):
        got = got.cpu().double()
        want = want.float().double()  # (below f32's range: -inf)
        same = got == want
        assert bool((same | ((got - want).abs() <= tol + want.abs() * 2.0 ** -22)).all()), (got, want)
    assert bool(((ent.cpu().double() - rent).abs() <= tol[:, 0] * (1 + math.log(vocab))).all()), (ent, rent)


def _tokens(rows, vocab, ids):
    g = torch.Generator().manual_seed(vocab)
    t = torch.randint(0, vocab, (rows, 4), generator=g).int()
    t[:, 0] = torch.as_tensor(ids).int()
    return t.cuda()


@pytest.mark.parametrize("ban", [-1e5, -1e9, -1e10, -1e30, -2.38e38, -2.9e38, LOWEST])
@pytest.mark.parametrize("vocab,allowed", [(70_001, 5), (262_144, 300), (5, 2), (4097, 4000)])
@pytest.mark.parametrize("cap", [0.0, 30.0, 1.0])
def test_logprobs_of_tokens_banned_by_a_finite_value(ctx, ban, vocab, allowed, cap):
    rows = 3
    g = torch.Generator().manual_seed(vocab)
    x = torch.full((rows, vocab), ban)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:allowed] for _ in range(rows)])
    x.scatter_(1, ids, torch.randn((rows, allowed), generator=g) * 4)
    x[2] = ban  # nothing but banned tokens: all equal
    _check(ctx, x.cuda(), _tokens(rows, vocab, ids[:, 0]), min(8, vocab), cap)


@pytest.mark.parametrize("ban", [-65504.0, -3e4])
def test_logprobs_of_f16_tokens_banned_by_the_lowest_value(ctx, ban):
    vocab = 50_257
    g = torch.Generator().manual_seed(1)
    x = torch.full((3, vocab), ban)
    x[0, 100:140] = torch.randn(40, generator=g)
    x[1, 50_000:] = torch.randn(257, generator=g) * 3 + 60_000
    _check(ctx, x.half().cuda(), _tokens(3, vocab, [101, 50_001, 7]), 8)


@pytest.mark.parametrize("top", [2000.0, 1e6, 1e30, 2.9e38, -LOWEST])
def test_logprobs_of_rows_with_a_huge_maximum(ctx, top):
    """The probability is the maximum's; with two of them a half each; differences beyond f32's range are -inf."""
    vocab = 20_000
    x = torch.randn((4, vocab), generator=torch.Generator().manual_seed(2)) * 3
    x[0, 9_999] = top
    x[1, 3], x[1, 19_998] = top, top
    x[2] = top
    x[3, :10_000], x[3, 15_000] = LOWEST, top
    _check(ctx, x.cuda(), _tokens(4, vocab, [9_999, 3, 11, 15_000]), 8)


@pytest.mark.parametrize("cap", [1024.0, 1500.0, 1e6])
def test_logprobs_under_a_large_cap(ctx, cap):
    """Caps on both sides of the size at which the exponents are formed in another way."""
    vocab = 30_011
    g = torch.Generator().manual_seed(3)
    x = torch.randn((4, vocab), generator=g) * 4
    x[1] += cap * 0.8
    x[2] -= cap * 3
    x[3, :29_000] = LOWEST
    _check(ctx, x.cuda(), _tokens(4, vocab, [9_999, 3, 11, 29_500]), 8, cap)


@pytest.mark.parametrize("cap", [1e-30, 1e-3, 30.0, 1e30])
def test_logprobs_under_the_smallest_and_largest_caps(ctx, cap):
    """An infinite logit is the cap's value, among finite ones."""
    vocab = 9_001
    x = torch.randn((2, vocab), generator=torch.Generator().manual_seed(4)) * 4
    x[1, 4_000] = math.inf
    x[1, 5_000] = 0.0
    _check(ctx, x.cuda(), _tokens(2, vocab, [9_000, 4_000]), 8, cap)
