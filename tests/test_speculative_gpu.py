"""The speculative-step operators over the paged cache against their 64-bit definitions.

f32 results are held to a few f32 roundings of the sums they come from, f16 results to one more
rounding of 2^-11 relative; tests/spec_ref.py derives the bounds.
"""
import math
import random

import numpy as np
import pytest
import torch

import g4attn
from g4attn import G4AError, gemma
from spec_ref import (Paged, logprob_ref, mask_tensor, prep_ref, seen_rows, tree_attn_ref, tree_masks,
                      tree_tolerance)

pytestmark = pytest.mark.gpu
EPS = 1e-6


# --------------------------------------------------------------------------------- rotation table

@pytest.mark.parametrize("hd,theta,div", [(256, 1e4, 0), (512, 1e6, 1), (64, 1e4, 0), (80, 1e4, 0)])
def test_rope_table_is_norm_ropes_rotation(ctx, hd, theta, div):
    pos = torch.tensor([0, 1, 2, 511, 4095, 131071, 1000003, -5], dtype=torch.int32)
    rf = torch.from_numpy(gemma.gemma_rope_freqs(hd).copy()) if div else None
    tab = torch.full((len(pos), hd), float("nan"), device="cuda")
    ctx.rope_table(pos.cuda(), None if rf is None else rf.cuda(), tab, head_dim=hd, theta=theta, apply_divisor=div)
    ctx.sync()
    p = np.arange(hd // 2)
    e = (2 * p).astype(np.float32) / np.float32(hd)
    freq = np.float32(1) / np.array([float(theta) ** float(x) for x in e]).astype(np.float32)
    if div:
        freq = freq / rf.numpy().astype(np.float32)
    ang = (np.maximum(pos.numpy(), 0).astype(np.float32)[:, None] * freq).astype(np.float32).astype(np.float64)
    want = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    got = tab.cpu().numpy()
    # the same f32 angle; cos and sin of it in doubles of two libraries, rounded once
    assert np.abs(got - want).max() <= 2.0 ** -24
    assert (got != want).mean() < 1e-3
    # and g4a_norm_rope turns by exactly these: a head whose pairs are (a, 0) shows cos and sin
    if hd % 2 == 0:
        w = torch.ones(hd, dtype=torch.float16, device="cuda")
        for i in (1, 4, 5):
            x = torch.zeros((1, hd), device="cuda")
            x[:, : hd // 2] = 1.0
            n = x.clone()
            ctx.norm_rope(n, w, None if rf is None else rf.cuda(), num_heads=1, head_dim=hd, eps=EPS,
                          position=int(pos[i]), theta=theta, apply_divisor=div)
            ctx.sync()
            a = np.float32(1) / np.float32(np.sqrt(np.float32(np.float32(0.5) + np.float32(EPS))))
            assert np.array_equal(n.cpu().numpy()[0], (got[i] * a).astype(np.float32))


# ------------------------------------------------------------------------------------ paged append

def _prep_case(seed, counts, starts, *, nqh, nkh, hd, page, fused=False, pad=0):
    g = torch.Generator().manual_seed(seed)
    n = sum(counts) + pad
    lens = [a + c for a, c in zip(starts, counts)]
    case = Paged(seed, lens, counts, nkh=nkh, hd=hd, page=page)
    width = (nqh + 2 * nkh) * hd
    whole = torch.randn((n, width), generator=g) * 2
    parts = list(whole.cuda().split([nqh * hd, nkh * hd, nkh * hd], 1))
    if not fused:
        parts = [p.contiguous() for p in parts]
    slots = [a + i for a, c in zip(starts, counts) for i in range(c)] + [0] * pad
    seq = [b for b, c in enumerate(counts) for _ in range(c)] + [-1] * pad
    ang = torch.rand((n, hd // 2), generator=g, dtype=torch.float64) * 6.3
    cs = torch.cat([ang.cos(), ang.sin()], 1).float().cuda()
    qw, kw = ((1 + 0.3 * torch.randn(hd, generator=g)).half().cuda() for _ in range(2))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return case, parts, i32(slots), i32(seq), cs, qw, kw, slots, seq


def _close(got, want, hd, f16):
    """Products of five f32 factors and a two-term sum (the norm's mean of hd values adds its own
    relative error, hd / 64 + 8 sums deep): 2^-24 * (hd / 64 + 16) of the pair's size."""
    h = want.shape[-1] // 2
    size = torch.sqrt(want[..., :h] ** 2 + want[..., h:] ** 2)
    size = torch.cat([size, size], -1) * 1.5
    tol = size * 2.0 ** -24 * (hd / 64 + 16) + (want.abs() * 2.0 ** -11 + 2.0 ** -24 if f16 else 0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-30)).max())


@pytest.mark.parametrize("hd,nqh,nkh", [(256, 8, 1), (512, 8, 1), (128, 12, 4), (64, 4, 4), (96, 6, 2), (8, 1, 1)])
@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("page,fused", [(64, True), (16, False), (5, True)])
def test_paged_prep_matches_definition(ctx, hd, nqh, nkh, fmt, page, fused):
    counts, starts = [1, 7, 40], [0, 13, 100]
    case, (q, k, v), slots, seq, cs, qw, kw, hslots, hseq = _prep_case(hd + page, counts, starts, nqh=nqh, nkh=nkh,
                                                                       hd=hd, page=page, fused=fused, pad=3)
    n = len(hseq)
    qo = torch.full((n, nqh, hd), 7.0, dtype=fmt, device="cuda")
    k0, v0 = case.k.clone(), case.v.clone()
    ctx.paged_qkv_prep(q, k, v, qw, kw, cs, qo, case.k, case.v, case.table, seq, slots, num_q_heads=nqh,
                       num_kv_heads=nkh, head_dim=hd, page_size=page, eps=EPS)
    ctx.sync()
    rq, rk, rv = prep_ref(q.cpu(), k.cpu(), v.cpu(), qw.cpu(), kw.cpu(), cs.cpu(), nqh, nkh, hd, EPS)
    live = n - 3
    _close(qo[:live], rq[:live], hd, fmt == torch.float16)
    assert bool((qo[live:] == 7.0).all())  # padding rows are left as they were
    touched = torch.zeros(k0.shape[:2], dtype=torch.bool)
    for i in range(live):
        pg, r = int(case.table_host[hseq[i], hslots[i] // page]), hslots[i] % page
        touched[pg, r] = True
        _close(case.k[pg, r], rk[i], hd, True)
        _close(case.v[pg, r], rv[i], hd, True)
    left = ~touched.cuda()
    for new, old in ((case.k, k0), (case.v, v0)):  # nothing else in the pool changed (NaN included)
        assert torch.equal(new[left].view(torch.int16), old[left].view(torch.int16))


def test_paged_prep_unaligned_rows_take_the_strided_instance(ctx):
    """Rows that start off a 16-byte boundary give the same values as aligned ones."""
    hd, nqh, nkh, n = 256, 8, 1, 9
    case, (q, k, v), slots, seq, cs, qw, kw, *_ = _prep_case(3, [n], [4], nqh=nqh, nkh=nkh, hd=hd, page=16)
    outs = []
    for shift in (0, 1):
        wide = [torch.zeros((n, x.shape[1] + 3 + shift), device="cuda") for x in (q, k, v)]
        views = [w[:, shift:shift + x.shape[1]] for w, x in zip(wide, (q, k, v))]
        for w, x in zip(views, (q, k, v)):
            w.copy_(x)
        qo = torch.zeros((n, nqh, hd), device="cuda")
        kp, vp = case.k.clone(), case.v.clone()
        ctx.paged_qkv_prep(*views, qw, kw, cs, qo, kp, vp, case.table, seq, slots, num_q_heads=nqh, num_kv_heads=nkh,
                           head_dim=hd, page_size=16, eps=EPS)
        ctx.sync()
        outs.append((qo, kp, vp))
    ref = prep_ref(q.cpu(), k.cpu(), v.cpu(), qw.cpu(), kw.cpu(), cs.cpu(), nqh, nkh, hd, EPS)[0]
    for qo, kp, vp in outs:
        _close(qo, ref, hd, False)
    assert torch.allclose(outs[0][1].float(), outs[1][1].float(), rtol=2 ** -10, atol=2 ** -20, equal_nan=True)


def test_paged_prep_consumer_layer_and_append_alone(ctx):
    hd, nqh, nkh = 256, 8, 2
    case, (q, k, v), slots, seq, cs, qw, kw, hslots, _ = _prep_case(5, [6], [30], nqh=nqh, nkh=nkh, hd=hd, page=8)
    rq, rk, _ = prep_ref(q.cpu(), k.cpu(), v.cpu(), qw.cpu(), kw.cpu(), cs.cpu(), nqh, nkh, hd, EPS)
    qo = torch.zeros((6, nqh, hd), device="cuda")
    k0 = case.k.clone()
    ctx.paged_qkv_prep(q, None, None, qw, None, cs, qo, case.k, case.v, case.table, seq, None, num_q_heads=nqh,
                       num_kv_heads=nkh, head_dim=hd, page_size=8, eps=EPS)
    ctx.sync()
    _close(qo, rq, hd, False)
    assert torch.equal(case.k.view(torch.int16), k0.view(torch.int16))
    some = slots.clone()
    some[2] = -1  # computed, not stored
    ctx.paged_qkv_prep(None, k, v, None, kw, cs, None, case.k, case.v, case.table, seq, some, num_q_heads=0,
                       num_kv_heads=nkh, head_dim=hd, page_size=8, eps=EPS)
    ctx.sync()
    for i, s in enumerate(hslots):
        pg, r = int(case.table_host[0, s // 8]), s % 8
        if i == 2:
            assert torch.equal(case.k[pg, r].view(torch.int16), k0[pg, r].view(torch.int16))
        else:
            _close(case.k[pg, r], rk[i], hd, True)


def test_paged_prep_reports_what_it_cannot_store(ctx):
    hd, nqh, nkh, page = 64, 2, 1, 8
    case, (q, k, v), slots, seq, cs, qw, kw, hslots, _ = _prep_case(6, [4, 4], [0, 0], nqh=nqh, nkh=nkh, hd=hd, page=page)
    rq, rk, _ = prep_ref(q.cpu(), k.cpu(), v.cpu(), qw.cpu(), kw.cpu(), cs.cpu(), nqh, nkh, hd, EPS)
    bad_slot, bad_seq, bad_table = slots.clone(), seq.clone(), case.table.clone()
    bad_slot[1] = 10 ** 6
    bad_seq[1] = 2
    bad_table[0, 0] = 999
    for s, sl, tb, what in ((seq, bad_slot, case.table, "slot"), (bad_seq, slots, case.table, "sequence index"),
                            (seq, slots, bad_table, "page id")):
        kp, vp = case.k.clone(), case.v.clone()
        qo = torch.full((8, nqh, hd), 3.0, device="cuda")
        ctx.paged_qkv_prep(q, k, v, qw, kw, cs, qo, kp, vp, tb, s, sl, num_q_heads=nqh, num_kv_heads=nkh, head_dim=hd,
                           page_size=page, eps=EPS)
        with pytest.raises(G4AError, match=what):
            ctx.sync()
        ctx.sync()
        _close(kp[int(case.table_host[1, 0]), 0], rk[4], hd, True)  # the other sequence is stored
        if what != "sequence index":
            _close(qo, rq, hd, False)
        else:
            assert bool((qo[1] == 3.0).all())


def test_paged_rows_agree_with_the_contiguous_producers(ctx):
    """The same token through g4a_prefill_qkv_prep and through the paged append: the same f16 rows up
    to the last bit of a rounding (the products are taken in another order)."""
    hd, nqh, nkh, n, theta = 256, 8, 1, 33, 1e4
    case, (q, k, v), slots, seq, _, qw, kw, hslots, _ = _prep_case(8, [n], [0], nqh=nqh, nkh=nkh, hd=hd, page=16)
    cs = torch.zeros((n, hd), device="cuda")
    ctx.rope_table(slots, None, cs, head_dim=hd, theta=theta)
    qo = torch.zeros((n, nqh, hd), dtype=torch.float16, device="cuda")
    ctx.paged_qkv_prep(q, k, v, qw, kw, cs, qo, case.k, case.v, case.table, seq, slots, num_q_heads=nqh,
                       num_kv_heads=nkh, head_dim=hd, page_size=16, eps=EPS)
    kc = torch.zeros((n, nkh, hd), dtype=torch.float16, device="cuda")
    vc, q16 = torch.zeros_like(kc), torch.zeros_like(qo)
    ctx.prefill_qkv_prep(q, k, v, qw, kw, None, q16, kc, vc, T=n, start_pos=0, max_seq_len=n, num_q_heads=nqh,
                         num_kv_heads=nkh, head_dim=hd, eps=EPS, theta=theta)
    ctx.sync()
    rows = case.table.long()[0, slots.long() // 16] * 16 + slots.long() % 16
    for a, b in ((qo, q16), (case.k.view(-1, nkh, hd)[rows], kc), (case.v.view(-1, nkh, hd)[rows], vc)):
        # one f16 step at most (2^-10 relative; below f16's normal range its smallest step), seldom
        assert bool(((a.double() - b.double()).abs() <= b.double().abs() * 2.0 ** -10 + 2.0 ** -24).all())
        assert float((a != b).double().mean()) < 0.01


# ---------------------------------------------------------------------------------- tree attention

def _run_tree(ctx, case, q, words, *, window=0, scale=None, host=True, extra=0, max_tokens=None):
    nqh, hd = q.shape[1], q.shape[2]
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device="cuda")
    ctx.tree_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr,
                        None if words is None else mask_tensor(words + [0] * extra), out, num_q_heads=nqh,
                        num_kv_heads=case.nkh, head_dim=hd, page_size=case.page,
                        max_tokens=max_tokens or max(max(case.counts), 1),
                        scale=hd ** -0.5 if scale is None else scale, sliding_window=window,
                        host_kv_lens=case.lens if host else None)
    return out


def _check_tree(out, case, q, words, *, window=0, scale=None):
    hd, n = q.shape[2], case.indptr_host[-1]
    ref, amp = tree_attn_ref(case, q[:n], words, scale=hd ** -0.5 if scale is None else scale, window=window)
    vmax = max((float(v.double().abs().max()) for _, v in case.rows if v.numel()), default=0.0)
    f16 = q.dtype == torch.float16
    tol = tree_tolerance(amp, hd, max(case.lens), vmax, f16)
    err = float((out[:n].double().cpu() - ref).abs().max()) if n else 0.0
    assert err <= tol, (err, tol)
    rel = float((out[:n].double().cpu() - ref).norm() / ref.norm().clamp_min(1e-30)) if n else 0.0
    # roundings of either sign: the norm of the error stays at the size of single roundings
    assert rel <= (2.0 ** -11 if f16 else 2.0 ** -23 * max(amp, 8.0)), rel
    assert bool((out[n:] == 5.0).all())  # rows behind the last sequence


@pytest.mark.parametrize("hd,nqh,nkh", [(256, 8, 1), (512, 8, 1), (128, 12, 4), (64, 4, 4), (96, 6, 2), (8, 3, 1)])
@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("kind,page,window", [("tree", 64, 0), ("chain", 16, 100), ("star", 5, 3), ("none", 48, 0)])
def test_tree_attn_matches_definition(ctx, hd, nqh, nkh, fmt, kind, page, window):
    rnd = random.Random(hd + page)
    counts = [1, 9, 0, 24, 5]
    lens = [1, 300, 17, 24, 1201]  # alone, prefix, no tokens, nothing but drafts, longer
    case = Paged(hd + page, lens, counts, nkh=nkh, hd=hd, page=page)
    words = None if kind == "none" else tree_masks(counts, rnd, kind)
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((sum(counts) + 2, nqh, hd), generator=g) * 2).to(fmt).cuda()
    for host in (True, False):
        out = _run_tree(ctx, case, q, words, window=window, host=host, extra=2)
        ctx.sync()
        _check_tree(out, case, q, words, window=window)


@pytest.mark.parametrize("T", [1, 2, 16, 33, 64])
@pytest.mark.parametrize("hd,fmt", [(256, torch.float32), (512, torch.float16), (512, torch.float32), (128, torch.float16)])
def test_tree_attn_sizes_of_trees(ctx, T, hd, fmt):
    rnd = random.Random(T)
    case = Paged(T + hd, [T + 777], [T], nkh=1, hd=hd, page=64)
    words = tree_masks([T], rnd)
    q = torch.randn((T, 8, hd), generator=torch.Generator().manual_seed(T)).to(fmt).cuda() * 2
    out = _run_tree(ctx, case, q, words)
    ctx.sync()
    _check_tree(out, case, q, words)


@pytest.mark.parametrize("window", [0, 1, 5, 64, 1000])
def test_tree_attn_windows_around_the_drafts(ctx, window):
    """Windows shorter than the tree's depth, ending in the prefix, and longer than everything."""
    counts, lens = [20, 20, 20], [20, 21, 400]
    case = Paged(window, lens, counts, nkh=1, hd=64, page=16)
    words = tree_masks(counts, random.Random(1), "chain")
    q = torch.randn((60, 8, 64), generator=torch.Generator().manual_seed(2)).cuda()
    out = _run_tree(ctx, case, q, words, window=window)
    ctx.sync()
    _check_tree(out, case, q, words, window=window)


def test_tree_attn_long_cache_split_over_all_sms(ctx):
    case = Paged(4, [20011, 3], [5, 3], nkh=1, hd=256, page=64)
    words = tree_masks([5, 3], random.Random(2))
    q = torch.randn((8, 8, 256), generator=torch.Generator().manual_seed(3)).cuda() * 3
    out = _run_tree(ctx, case, q, words)
    ctx.sync()
    _check_tree(out, case, q, words)


@pytest.mark.parametrize("hd,nqh,nkh,fmt,T,n", [(256, 8, 1, torch.float32, 48, 9001), (512, 8, 1, torch.float16, 40, 6007),
                                                (128, 12, 4, torch.float32, 64, 5000), (256, 8, 1, torch.float16, 64, 4100),
                                                (512, 4, 1, torch.float32, 20, 3001)])
def test_tree_attn_several_tiles_over_a_long_cache(ctx, hd, nqh, nkh, fmt, T, n):
    """Every tile's keys are cut into several pieces, and the pieces of several tiles are joined."""
    case = Paged(n, [n], [T], nkh=nkh, hd=hd, page=64)
    words = tree_masks([T], random.Random(n))
    q = (torch.randn((T, nqh, hd), generator=torch.Generator().manual_seed(n)) * 2).to(fmt).cuda()
    for window in (0, n // 2):
        out = _run_tree(ctx, case, q, words, window=window)
        ctx.sync()
        _check_tree(out, case, q, words, window=window)


@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("batch,longest,nkh,group,most", [
    (60, 900, 4, 2, 8),   # more tiles than SMs: tiles cut at any stage, two pieces to a CTA
    (9, 6000, 2, 8, 24),  # short sequences beside one that is far longer than the rest
    (33, 500, 1, 8, 5),   # just past 32 sequences
    (600, 90, 1, 4, 3),   # more sequences than the table in shared memory holds
])
def test_tree_attn_partitions(ctx, fmt, batch, longest, nkh, group, most):
    rnd = random.Random(batch)
    counts = [rnd.randint(0, most) for _ in range(batch)]
    counts[0], counts[-1] = most, max(counts[-1], 1)
    lens = [c + (rnd.randint(0, longest) if batch != 9 or b == 4 else rnd.randint(0, 60)) for b, c in enumerate(counts)]
    lens[batch // 2] = longest
    case = Paged(batch, lens, counts, nkh=nkh, hd=64, page=16)
    words = tree_masks(counts, rnd)
    g = torch.Generator().manual_seed(batch)
    q = (torch.randn((sum(counts) + 1, nkh * group, 64), generator=g) * 2).to(fmt).cuda()
    for host, window in ((True, 0), (False, 0), (True, 200)):
        out = _run_tree(ctx, case, q, words, window=window, host=host, extra=1)
        ctx.sync()
        _check_tree(out, case, q, words, window=window)


@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
def test_tree_attn_empty_masks_give_zeros(ctx, fmt):
    """A word without bits sees the prefix alone; without a prefix it sees nothing and gives zeros."""
    case = Paged(1, [4, 10], [4, 4], nkh=1, hd=128, page=16)
    words = [0, 1, 0, 8, 0, 3, 0, 8]
    q = torch.randn((8, 8, 128), generator=torch.Generator().manual_seed(3)).to(fmt).cuda()
    for window in (0, 4):
        out = _run_tree(ctx, case, q, words, window=window)
        ctx.sync()
        assert not out[0].any() and not out[2].any()
        _check_tree(out, case, q, words, window=window)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hd,fmt,T", [(256, torch.float32, 8), (512, torch.float16, 8), (128, torch.float32, 8),
                                      (256, torch.float16, 40), (64, torch.float32, 40), (512, torch.float32, 40)])
def test_tree_attn_non_finite_rows_reach_only_their_observers(ctx, what, hd, fmt, T):
    """K and V of one drafted token (and of a prefix row outside some windows) are not finite."""
    case = Paged(9, [90 + T], [T], nkh=1, hd=hd, page=16)
    words = [1 << i for i in range(T)]  # every token sees itself alone
    q = torch.randn((T, 8, hd), generator=torch.Generator().manual_seed(4)).to(fmt).cuda()
    good = _run_tree(ctx, case, q, words)
    ctx.sync()
    s = 90 + 3
    pg, r = int(case.table_host[0, s // 16]), s % 16
    case.k[pg, r] = what
    case.v[pg, r] = what
    out = _run_tree(ctx, case, q, words)
    ctx.sync()
    hit = torch.zeros(T, dtype=torch.bool)
    hit[3] = True
    assert not bool(torch.isfinite(out[3].float()).any())
    # the others keep their values: to the rounding of p (f16: the stage is summed in f32 then)
    assert bool(torch.isfinite(out[~hit].float()).all())
    assert float((out[~hit].double() - good[~hit].double()).abs().max()) <= 2.0 ** -10 * float(good.abs().max())


def test_tree_attn_large_and_small_queries(ctx):
    """Queries far from 1 keep their accuracy: rows scaled by 2^40 and 2^-40 against scales that undo it."""
    case = Paged(3, [200], [6], nkh=1, hd=256, page=64)
    words = tree_masks([6], random.Random(3))
    q = torch.randn((6, 8, 256), generator=torch.Generator().manual_seed(5)).cuda()
    for e in (-40, 0, 40):
        qq = q * 2.0 ** e
        out = _run_tree(ctx, case, qq, words, scale=2.0 ** (-4 - e))
        ctx.sync()
        _check_tree(out, case, qq, words, scale=2.0 ** (-4 - e))


def test_tree_attn_agrees_with_decode(ctx):
    """One new token per sequence is g4a_decode_attn_paged."""
    lens = [1, 513, 2000]
    case = Paged(12, lens, [1, 1, 1], nkh=1, hd=256, page=64)
    q = torch.randn((3, 8, 256), generator=torch.Generator().manual_seed(6)).cuda() * 2
    for window in (0, 512):
        out = _run_tree(ctx, case, q, None, window=window)
        dec = torch.zeros_like(out)
        ctx.decode_attn_paged(q, torch.nan_to_num(case.k), torch.nan_to_num(case.v), case.table, case.lens_dev, dec,
                              num_q_heads=8, num_kv_heads=1, head_dim=256, page_size=64, scale=256 ** -0.5,
                              sliding_window=window, host_kv_lens=lens)
        ctx.sync()
        assert float((out - dec).abs().max()) <= 2 * tree_tolerance(16.0, 256, 2000, 4.5, False)


def test_tree_attn_is_reproducible_and_independent_of_neighbours(ctx):
    case = Paged(13, [900, 50], [12, 3], nkh=1, hd=256, page=64)
    words = tree_masks([12, 3], random.Random(5))
    q = torch.randn((15, 8, 256), generator=torch.Generator().manual_seed(7)).cuda()
    a = _run_tree(ctx, case, q, words)
    b = _run_tree(ctx, case, q, words)
    ctx.sync()
    assert torch.equal(a, b)


def test_tree_attn_reports_sequences_that_do_not_fit(ctx):
    counts, lens = [3, 4, 5], [30, 40, 50]
    case = Paged(14, lens, counts, nkh=1, hd=64, page=16)
    q = torch.randn((12, 8, 64), generator=torch.Generator().manual_seed(8)).cuda()
    good = _run_tree(ctx, case, q, None)
    ctx.sync()
    cases = []
    short = case.lens_dev.clone()
    short[1] = 2  # fewer rows than tokens
    cases.append(dict(kv_lens=short, q_indptr=case.indptr, max_tokens=5, bad=[1]))
    over = case.lens_dev.clone()
    over[2] = 16 * case.table.shape[1] + 1
    cases.append(dict(kv_lens=over, q_indptr=case.indptr, max_tokens=5, bad=[2]))
    cases.append(dict(kv_lens=case.lens_dev, q_indptr=case.indptr, max_tokens=4, bad=[2]))
    wild = case.indptr.clone()
    wild[3] = 13  # behind the last row
    cases.append(dict(kv_lens=case.lens_dev, q_indptr=wild, max_tokens=8, bad=[2]))
    for c in cases:
        out = torch.full_like(q, 5.0)
        ctx.tree_attn_paged(q, case.k, case.v, case.table, c["kv_lens"], c["q_indptr"], None, out, num_q_heads=8,
                            num_kv_heads=1, head_dim=64, page_size=16, max_tokens=c["max_tokens"], scale=64 ** -0.5)
        with pytest.raises(G4AError, match="q_indptr and kv_lens"):
            ctx.sync()
        ctx.sync()
        for b in range(3):
            i0, i1 = case.indptr_host[b], case.indptr_host[b + 1]
            if b in c["bad"]:
                assert bool((out[i0:i1] == 5.0).all())
            else:
                assert float((out[i0:i1] - good[i0:i1]).abs().max()) <= 2.0 ** -19


def test_tree_attn_bad_page_rows_are_not_there(ctx):
    case = Paged(15, [100], [4], nkh=1, hd=128, page=16)
    q = torch.randn((4, 8, 128), generator=torch.Generator().manual_seed(9)).cuda()
    for bad in (10 ** 6, -1):
        table = case.table.clone()
        table[0, 2] = bad  # rows 32..47
        out = torch.zeros_like(q)
        ctx.tree_attn_paged(q, case.k, case.v, table, case.lens_dev, case.indptr, None, out, num_q_heads=8,
                            num_kv_heads=1, head_dim=128, page_size=16, max_tokens=4, scale=128 ** -0.5)
        with pytest.raises(G4AError, match="page id"):
            ctx.sync()
        ctx.sync()
        k, v = (x[:, 0].double() for x in case.rows[0])
        for i in range(4):
            r = torch.tensor([x for x in range(97 + i) if not 32 <= x < 48])
            for h in range(8):
                s = torch.softmax(k[r] @ q[i, h].double().cpu() * 128 ** -0.5, 0)
                assert float((out[i, h].double().cpu() - s @ v[r]).abs().max()) <= tree_tolerance(24.0, 128, 100, 4.5, False)


def test_tree_attn_offsets_beyond_32_bits(ctx):
    """Pages whose element offsets pass 2^31 (a pool of more than 4 GiB)."""
    hd, page, per = 512, 64, 64 * 512
    far = 2 ** 31 // per + 5
    small = Paged(16, [150], [3], nkh=1, hd=hd, page=page)
    k = torch.empty((far + 8, page, 1, hd), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    where = torch.tensor([far + 7, 1, far], dtype=torch.int32, device="cuda")
    for j in range(3):
        k[int(where[j])] = small.k[int(small.table_host[0, j])]
        v[int(where[j])] = small.v[int(small.table_host[0, j])]
    q = torch.randn((3, 8, hd), generator=torch.Generator().manual_seed(10)).cuda()
    out = torch.zeros_like(q)
    ctx.tree_attn_paged(q, k, v, where[None].contiguous(), small.lens_dev, small.indptr, None, out, num_q_heads=8,
                        num_kv_heads=1, head_dim=hd, page_size=page, max_tokens=3, scale=hd ** -0.5)
    ctx.sync()
    _check_tree(out, small, q, None)
    # and the move of rows there
    base = torch.tensor([140], dtype=torch.int32, device="cuda")
    path = torch.tensor([[3, 9]], dtype=torch.int32, device="cuda")
    n = torch.tensor([2], dtype=torch.int32, device="cuda")
    src = [k[far, (140 + j) % 64].clone() for j in (3, 9)]
    ctx.paged_kv_compact(k, v, where[None].contiguous(), base, path, n, num_kv_heads=1, head_dim=hd, page_size=page)
    ctx.sync()
    assert torch.equal(k[far, 12], src[0]) and torch.equal(k[far, 13], src[1])


# ------------------------------------------------------------------------------- log probabilities

def _run_logprobs(ctx, x, tokens, k, cap):
    rows = x.shape[0]
    lp = torch.full((rows, tokens.shape[1]), 9.0, device="cuda")
    ent = torch.full((rows,), 9.0, device="cuda")
    tv = torch.full((rows, k), 9.0, device="cuda")
    ti = torch.full((rows, k), -9, dtype=torch.int32, device="cuda")
    ctx.token_logprobs(x, tokens, lp, ent, tv, ti, softcap=cap)
    return lp, ent, tv, ti


def _check_logprobs(got, x, tokens, k, cap):
    """A logit's own f32 size sets the scale: y, its maximum and log Z each within 2^-22 of it (the
    capped logit 2^-21: four roundings), sums of vocab f32 terms 2^-20 relative (in 4096-value tiles)."""
    lp, ent, tv, ti = (t.cpu() for t in got)
    rlp, rent, rtv, rti = logprob_ref(x.cpu(), tokens.cpu(), k, cap)
    assert torch.equal(ti.long(), rti)
    fin = x[torch.isfinite(x)]
    size = max(float(fin.abs().max()) if fin.numel() else 1.0, 1.0)
    if cap:
        size = min(size, cap) + cap
    tol = size * 2.0 ** -21 + 2.0 ** -20
    for a, b in ((lp, rlp), (ent, rent), (tv, rtv)):
        if not a.numel():
            continue
        a = a.double()
        same = (a == b) | (torch.isnan(a) & torch.isnan(b))
        err = torch.where(same, 0.0, (a - b).abs())
        # entropy also sums sum p |y - m|: relative 2^-20 of itself
        assert bool((err <= tol + b.abs() * 2.0 ** -19).all()), (float(err.max()), tol)


@pytest.mark.parametrize("vocab", [1, 31, 4095, 4097, 50257, 262144])
@pytest.mark.parametrize("rows,fmt,cap,k", [(1, torch.float32, 30.0, 20), (3, torch.float16, 0.0, 5),
                                            (150, torch.float32, 0.0, 1), (7, torch.float16, 30.0, 32), (2, torch.float32, 0.0, 0)])
def test_logprobs_match_definition(ctx, vocab, rows, fmt, cap, k):
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = (torch.randn((rows, vocab), generator=g, device="cuda") * 4).to(fmt)
    tokens = torch.randint(-1, vocab, (rows, 3), generator=g, device="cuda").int()
    tokens[0, 0] = -1
    got = _run_logprobs(ctx, x, tokens, min(k, vocab), cap)
    ctx.sync()
    _check_logprobs(got, x, tokens, min(k, vocab), cap)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two", "peak", "banned", "zeros", "all_banned"])
@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_logprobs_hard_orders(ctx, kind, fmt, cap):
    """Ties, sorted rows, a single peak, banned tokens: the bounded candidate lists still hold."""
    vocab, k = 70001, 32
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    x = {"equal": torch.full_like(i, 2.5), "rising": i / 2000, "falling": -i / 2000, "two": (i % 2) * 3.0,
         "peak": torch.where(i == 69999, 40.0, -5.0), "banned": torch.where(i % 1000 == 7, i / 10000, -math.inf),
         "zeros": torch.where(i % 3 == 0, 0.0, -0.0), "all_banned": torch.full_like(i, -math.inf)}[kind]
    x = torch.stack([x, x.flip(0)]).to(fmt)
    tokens = torch.tensor([[0, 7, 69999], [1, 2, 3]], dtype=torch.int32, device="cuda")
    got = _run_logprobs(ctx, x, tokens, k, cap)
    ctx.sync()
    if kind == "all_banned":  # nothing to distribute: NaN, and the first ids
        assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[1]).all())
        assert torch.equal(got[3].cpu(), torch.arange(k).int().expand(2, k))
        return
    _check_logprobs(got, x, tokens, k, cap)


def test_logprobs_nan_and_inf_rows(ctx):
    x = torch.randn((4, 9000), generator=torch.Generator().manual_seed(1)).cuda()
    x[1, 5000] = float("nan")
    x[2, 17] = float("inf")
    tokens = torch.tensor([[3], [3], [3], [3]], dtype=torch.int32, device="cuda")
    lp, ent, tv, ti = _run_logprobs(ctx, x, tokens, 4, 0.0)
    ctx.sync()
    for r in (1, 2):
        assert bool(torch.isnan(lp[r]).all()) and bool(torch.isnan(ent[r]))
    assert int(ti[2, 0]) == 17 and 5000 not in ti[1].tolist()
    clean = x[[0, 3]]
    _check_logprobs((lp[[0, 3]], ent[[0, 3]], tv[[0, 3]], ti[[0, 3]]), clean, tokens[:2], 4, 0.0)


def test_logprobs_strides_alignment_and_parts_left_out(ctx):
    g = torch.Generator().manual_seed(2)
    for fmt in (torch.float32, torch.float16):
        wide = (torch.randn((5, 5011), generator=g) * 3).to(fmt).cuda()
        for a in (0, 1, 3):
            x = wide[:, a:a + 4999]
            tokens = torch.tensor([[0], [1], [4998], [77], [-1]], dtype=torch.int32, device="cuda")
            got = _run_logprobs(ctx, x, tokens, 7, 0.0)
            ctx.sync()
            _check_logprobs(got, x, tokens, 7, 0.0)
    x = wide[:, :4999]
    ent = torch.zeros(5, device="cuda")
    ctx.token_logprobs(x, None, None, ent)
    lp = torch.zeros(5, device="cuda")
    ctx.token_logprobs(x, tokens[:, 0].contiguous(), lp)
    tv, ti = torch.zeros((5, 7), device="cuda"), torch.zeros((5, 7), dtype=torch.int32, device="cuda")
    ctx.token_logprobs(x, None, None, None, tv, ti)
    ctx.sync()
    for a, b in ((ent, got[1]), (tv, got[2]), (ti, got[3])):
        full = _run_logprobs(ctx, x, tokens, 7, 0.0)
        ctx.sync()
        assert torch.equal(a, full[{id(ent): 1, id(tv): 2, id(ti): 3}[id(a)]])
    assert torch.equal(lp[:, None], full[0])


def test_logprobs_rows_beyond_32_bit_offsets(ctx):
    vocab = 5000
    flat = torch.empty(2 ** 31 + 4 * vocab, dtype=torch.float16, device="cuda")
    x = flat.as_strided((2, vocab), (2 ** 31 + 8, 1))
    x.copy_((torch.randn((2, vocab), generator=torch.Generator().manual_seed(3)) * 3).half())
    tokens = torch.tensor([[1], [4999]], dtype=torch.int32, device="cuda")
    got = _run_logprobs(ctx, x, tokens, 3, 0.0)
    ctx.sync()
    _check_logprobs(got, x.contiguous(), tokens, 3, 0.0)


def test_logprobs_reports_tokens_beyond_the_vocabulary(ctx):
    x = torch.randn((2, 100), generator=torch.Generator().manual_seed(4)).cuda()
    tokens = torch.tensor([[100, 5], [-2, 6]], dtype=torch.int32, device="cuda")
    lp, *_ = _run_logprobs(ctx, x, tokens, 0, 0.0)
    with pytest.raises(G4AError, match="vocabulary"):
        ctx.sync()
    ctx.sync()
    assert bool(torch.isnan(lp[:, 0]).all()) and bool(torch.isfinite(lp[:, 1]).all())


# -------------------------------------------------------------------------------------- compaction

@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
def test_logprobs_of_vocabularies_of_more_than_1024_segments(ctx, fmt):
    """More than 524,288 ids: the join goes through the segments tile by tile."""
    rows, vocab, k = 2, 600_001, 32
    g = torch.Generator().manual_seed(rows)
    logits = (torch.randn((rows, vocab), generator=g) * 4).to(fmt).cuda()
    toks = torch.randint(vocab, (rows, 3), generator=g).int().cuda()
    for cap in (0.0, 30.0):
        got = _run_logprobs(ctx, logits, toks, k, cap)
        ctx.sync()
        _check_logprobs(got, logits, toks, k, cap)


@pytest.mark.parametrize("nkh,hd,page", [(1, 256, 64), (4, 128, 16), (2, 8, 3), (1, 512, 7)])
def test_compact_moves_rows_as_if_read_first(ctx, nkh, hd, page):
    rnd = random.Random(hd)
    base = [0, 5, 130, 64]
    case = Paged(hd, [b + 64 for b in base], [64] * 4, nkh=nkh, hd=hd, page=page)
    # shifted by one (every source is the next one's target), reversed, scattered, and nothing
    paths = [list(range(1, 64)) + [0], list(range(63, 31, -1)), sorted(rnd.sample(range(64), 20)), []]
    path = torch.full((4, 64), -7, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    k0, v0 = case.k.clone(), case.v.clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ctx.paged_kv_compact(case.k, case.v, case.table, i32(base), path.cuda(), i32([len(p) for p in paths]),
                         num_kv_heads=nkh, head_dim=hd, page_size=page)
    ctx.sync()
    wk, wv = k0.clone(), v0.clone()
    for b, p in enumerate(paths):
        at = lambda s: (int(case.table_host[b, s // page]), s % page)  # noqa: E731, B023
        for i, j in enumerate(p):
            wk[at(base[b] + i)] = k0[at(base[b] + j)]
            wv[at(base[b] + i)] = v0[at(base[b] + j)]
    assert torch.equal(case.k.view(torch.int16), wk.view(torch.int16))
    assert torch.equal(case.v.view(torch.int16), wv.view(torch.int16))


def test_compact_reports_and_skips_what_is_out_of_range(ctx):
    case = Paged(2, [40, 40], [8, 8], nkh=1, hd=64, page=8)
    k0 = case.k.clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    path = i32([[5, 1000, 6], [2, 3, -4]])
    for lens, match in (([3, 3], "path entry"), ([4, 3], "path entry")):
        case.k.copy_(k0)
        ctx.paged_kv_compact(case.k, case.v, case.table, i32([30, 30]), path, i32(lens), num_kv_heads=1, head_dim=64,
                             page_size=8)
        with pytest.raises(G4AError, match=match):
            ctx.sync()
        ctx.sync()
        at = lambda b, s: (int(case.table_host[b, s // 8]), s % 8)  # noqa: E731
        first = k0[at(0, 35)] if lens[0] == 3 else k0[at(0, 30)]
        assert torch.equal(case.k[at(0, 30)].view(torch.int16), first.view(torch.int16))
        assert torch.equal(case.k[at(0, 31)].view(torch.int16), k0[at(0, 31)].view(torch.int16))
        assert torch.equal(case.k[at(1, 30)], k0[at(1, 32)]) and torch.equal(case.k[at(1, 32)], k0[at(1, 32)])


# --------------------------------------------------------------------- streams, graphs, a whole step

def test_other_streams_and_contexts(ctx):
    """A second context on its own stream gives the same bits while the first one works."""
    case = Paged(20, [700], [9], nkh=1, hd=256, page=64)
    words = tree_masks([9], random.Random(6))
    q = torch.randn((9, 8, 256), generator=torch.Generator().manual_seed(11)).cuda()
    want = _run_tree(ctx, case, q, words)
    ctx.sync()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with g4attn.Context(0) as other:
        other.set_stream(side.cuda_stream)
        b = []
        for _ in range(3):
            o = torch.zeros_like(q)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                other.tree_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, mask_tensor(words), o,
                                      num_q_heads=8, num_kv_heads=1, head_dim=256, page_size=64, max_tokens=9,
                                      scale=256 ** -0.5)
            b.append(o)
        mine = _run_tree(ctx, case, q, words)
        ctx.sync()
        other.sync()
        assert torch.equal(mine, want) and all(torch.equal(x, want) for x in b)


def test_capture_and_replay_a_step(ctx):
    """A captured step (append, attention, log probabilities, move) replays on changed inputs; growing
    the workspace afterwards does not disturb it, and growth inside a capture is refused."""
    hd, nqh, nkh, page, T = 256, 8, 1, 16, 6
    case = Paged(21, [100 + T], [T], nkh=nkh, hd=hd, page=page)
    words = tree_masks([T], random.Random(7))
    mask = mask_tensor(words)
    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn((T, n * hd), generator=g).cuda() for n in (nqh, nkh, nkh))
    qw = torch.ones(hd, dtype=torch.float16, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    slots, seq, pos = i32(list(range(100, 100 + T))), i32([0] * T), i32([100] * T)
    cs, qo, out = torch.zeros((T, hd), device="cuda"), torch.zeros((T, nqh, hd), device="cuda"), torch.zeros((T, nqh, hd), device="cuda")
    logits = torch.randn((T, 3001), generator=g).cuda()
    tokens, lp = i32([[i] for i in range(T)]), torch.zeros((T, 1), device="cuda")
    base, path, plen = i32([100]), i32([[0, 3, 5]]), i32([3])

    def step(c):
        c.rope_table(pos, None, cs, head_dim=hd, theta=1e4)
        c.paged_qkv_prep(q, k, v, qw, qw, cs, qo, case.k, case.v, case.table, seq, slots, num_q_heads=nqh,
                         num_kv_heads=nkh, head_dim=hd, page_size=page, eps=EPS)
        c.tree_attn_paged(qo, case.k, case.v, case.table, case.lens_dev, case.indptr, mask, out, num_q_heads=nqh,
                          num_kv_heads=nkh, head_dim=hd, page_size=page, max_tokens=T)
        c.token_logprobs(logits, tokens, lp)
        c.paged_kv_compact(case.k, case.v, case.table, base, path, plen, num_kv_heads=nkh, head_dim=hd, page_size=page)

    side = torch.cuda.Stream()
    with g4attn.Context(0) as c:
        c.set_stream(side.cuda_stream)
        with pytest.raises(G4AError, match="before capturing"):
            torch.cuda.synchronize()
            bad = torch.cuda.CUDAGraph()
            with torch.cuda.graph(bad, stream=side):
                c.tree_attn_paged(qo, case.k, case.v, case.table, case.lens_dev, case.indptr, mask, out,
                                  num_q_heads=nqh, num_kv_heads=nkh, head_dim=hd, page_size=page, max_tokens=T)
        torch.cuda.synchronize()
        step(c)
        c.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(c)
        for rep in range(2):
            q.copy_(torch.randn(q.shape, generator=g))
            logits.copy_(torch.randn(logits.shape, generator=g))
            torch.cuda.synchronize()
            if rep == 1:  # outgrow the workspace the graph was captured with
                c.reserve_workspace(512, 512, 64)
            graph.replay()
            torch.cuda.synchronize()
            got, got_lp = out.clone(), lp.clone()
            out.zero_()
            lp.zero_()
            torch.cuda.synchronize()
            step(c)
            c.sync()
            assert torch.equal(got, out) and torch.equal(got_lp, lp) and bool(got.any())
        del graph


@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
def test_captured_tree_attention_follows_lengths_pages_and_masks(ctx, fmt):
    """One graph, captured while the sequences were short, replayed for longer, shorter and empty ones on
    other pages: the partition is found from what is on the device at replay."""
    cases = [Paged(30 + i, lens, counts, nkh=1, hd=128, page=16, spare=1) for i, (lens, counts) in enumerate(
        [([40, 30, 20], [4, 3, 2]), ([2500, 6, 900], [5, 2, 2]), ([0, 1, 700], [0, 1, 8]), ([8, 0, 0], [8, 0, 0])])]
    pages, width = max(c.k.shape[0] for c in cases), max(c.table.shape[1] for c in cases)
    k = torch.zeros((pages, 16, 1, 128), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.zeros((3, width), dtype=torch.int32, device="cuda")
    lens, indptr = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    mask = torch.zeros(9, dtype=torch.int64, device="cuda")
    q, out = torch.zeros((9, 8, 128), dtype=fmt, device="cuda"), torch.zeros((9, 8, 128), dtype=fmt, device="cuda")

    def load(case, words, x):
        k[:case.k.shape[0]], v[:case.v.shape[0]] = case.k, case.v
        table.zero_()
        table[:, :case.table.shape[1]] = case.table
        lens.copy_(case.lens_dev)
        indptr.copy_(case.indptr)
        mask.zero_()
        mask[:len(words)] = mask_tensor(words)
        q.copy_(x)
        out.fill_(5.0)
        torch.cuda.synchronize()

    g = torch.Generator().manual_seed(31)
    side = torch.cuda.Stream()
    with g4attn.Context(0) as c:
        c.set_stream(side.cuda_stream)
        run = lambda: c.tree_attn_paged(q, k, v, table, lens, indptr, mask, out, num_q_heads=8, num_kv_heads=1,  # noqa: E731
                                        head_dim=128, page_size=16, max_tokens=8, scale=128 ** -0.5,
                                        host_kv_lens=cases[0].lens)
        graph = None
        for case in cases:
            words = tree_masks(case.counts, random.Random(31))
            x = (torch.randn((9, 8, 128), generator=g) * 2).to(fmt)
            load(case, words, x)
            if graph is None:
                run()
                c.sync()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    run()
            out.fill_(5.0)
            torch.cuda.synchronize()
            graph.replay()
            c.sync()
            torch.cuda.synchronize()
            _check_tree(out, case, x.cuda(), words)
        del graph


def test_speculative_step_equals_decoding_one_by_one(ctx):
    """A whole step for two sequences: prompt chunk into the pages, a drafted tree, attention of all
    its tokens at once, the accepted path moved together, and the next token decoded from the pages.
    Every tree token's attention equals decoding that token alone after its ancestors."""
    hd, nqh, nkh, page, theta, window = 256, 8, 1, 16, 1e4, 40
    g = torch.Generator().manual_seed(13)
    rnd = random.Random(8)
    prompt, T = [37, 90], [7, 5]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cap = [-(-(p + 64) // page) for p in prompt]
    table = torch.zeros((2, max(cap)), dtype=torch.int32)
    order = torch.randperm(sum(cap), generator=g).int()
    table[0, :cap[0]], table[1, :cap[1]] = order[:cap[0]], order[cap[0]:]
    kp = torch.zeros((sum(cap), page, nkh, hd), dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    qw, kw = ((1 + 0.1 * torch.randn(hd, generator=g)).half().cuda() for _ in range(2))
    tab = table.cuda()

    def append(seq, slots, positions, qkv):
        n = len(seq)
        cs = torch.zeros((n, hd), device="cuda")
        ctx.rope_table(i32(positions), None, cs, head_dim=hd, theta=theta)
        qo = torch.zeros((n, nqh, hd), device="cuda")
        q, k, v = qkv.split([nqh * hd, hd, hd], 1)
        ctx.paged_qkv_prep(q, k, v, qw, kw, cs, qo, kp, vp, tab, i32(seq), i32(slots), num_q_heads=nqh,
                           num_kv_heads=nkh, head_dim=hd, page_size=page, eps=EPS)
        return qo

    rand = lambda n: torch.randn((n, (nqh + 2) * hd), generator=g).cuda()  # noqa: E731
    append([b for b in (0, 1) for _ in range(prompt[b])], [i for b in (0, 1) for i in range(prompt[b])],
           [i for b in (0, 1) for i in range(prompt[b])], rand(sum(prompt)))
    words = tree_masks(T, rnd)
    depth = [bin(w).count("1") - 1 for w in words]
    seq = [0] * T[0] + [1] * T[1]
    node = list(range(T[0])) + list(range(T[1]))
    tree_qkv = rand(sum(T))
    positions = [prompt[b] + d for b, d in zip(seq, depth)]
    q_tree = append(seq, [prompt[b] + j for b, j in zip(seq, node)], positions, tree_qkv)
    out = torch.zeros_like(q_tree)
    lens = [p + t for p, t in zip(prompt, T)]
    ctx.tree_attn_paged(q_tree, kp, vp, tab, i32(lens), i32([0, T[0], sum(T)]), mask_tensor(words), out,
                        num_q_heads=nqh, num_kv_heads=nkh, head_dim=hd, page_size=page, max_tokens=max(T),
                        sliding_window=window, host_kv_lens=lens)
    ctx.sync()
    # each token alone: its ancestors moved behind the prompt in a copy of the cache, then decode
    tol = 2 * tree_tolerance(256 * 2.0, hd, 100, 5.0, False)
    for r, w in enumerate(words):
        b = seq[r]
        mine = [j for j in range(64) if w >> j & 1]
        k2, v2 = kp.clone(), vp.clone()
        path = torch.full((2, 64), 0, dtype=torch.int32)
        path[b, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        ctx.paged_kv_compact(k2, v2, tab, i32(prompt), path.cuda(), i32([len(mine) if x == b else 0 for x in (0, 1)]),
                             num_kv_heads=nkh, head_dim=hd, page_size=page)
        dec = torch.zeros((2, nqh, hd), device="cuda")
        kl = [prompt[x] + (len(mine) if x == b else 0) for x in (0, 1)]
        qq = torch.zeros((2, nqh, hd), device="cuda")
        qq[b] = q_tree[r]
        ctx.decode_attn_paged(qq, k2, v2, tab, i32(kl), dec, num_q_heads=nqh, num_kv_heads=nkh, head_dim=hd,
                              page_size=page, sliding_window=window, host_kv_lens=kl)
        ctx.sync()
        assert float((dec[b] - out[r]).abs().max()) <= tol, r
    # the drafts' probabilities under (random) target logits pick a path; its rows are then in place
    vocab = 1000
    logits = torch.randn((sum(T), vocab), generator=g).cuda()
    toks = torch.randint(vocab, (sum(T), 2), generator=g).int().cuda()
    got = _run_logprobs(ctx, logits, toks, 3, 30.0)
    ctx.sync()
    _check_logprobs(got, logits, toks, 3, 30.0)


def test_profiler_labels_of_the_step(ctx):
    case = Paged(22, [300], [4], nkh=1, hd=128, page=16)
    q = torch.randn((4, 8, 128), generator=torch.Generator().manual_seed(14)).cuda()
    ctx.profile_enable(True)
    ctx.profile_reset()
    _run_tree(ctx, case, q, None)
    ms, n = ctx.profile_read("tree_attn")
    ctx.profile_enable(False)
    assert n == 1 and ms > 0
