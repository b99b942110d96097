"""Chunk attention with sinks, key masses and eviction over the paged cache against their 64-bit definitions; the bounds
are derived in tests/chunk_ref.py."""
import random

import pytest
import torch

import g4attn
from chunk_ref import attn_tolerance, chunk_ref, evict_ref, lse_tolerance, mass_ref, mass_tolerance
from g4attn import G4AError
from spec_ref import Paged

pytestmark = pytest.mark.gpu


def _case(seed, counts, lens, *, nkh, group, hd, page, spread=3.0):
    case = Paged(seed, lens, counts, nkh=nkh, hd=hd, page=page)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((sum(counts), nkh * group, hd), generator=g) * spread).half().cuda()
    return case, q


def _shape(case, q):
    return dict(num_q_heads=q.shape[1], num_kv_heads=case.nkh, head_dim=q.shape[2], page_size=case.page)


def _attend(ctx, case, q, *, window=0, sinks=0, scale=None, tail=3, sync=True):
    """out and lse of the call, with `tail` rows behind the last sequence that have to stay as they were."""
    n, nqh, hd = q.shape
    qq = torch.cat([q, torch.full((tail, nqh, hd), float("nan"), dtype=q.dtype, device="cuda")])
    out, lse = torch.full_like(qq, 7.0), torch.full((n + tail, nqh), 7.0, device="cuda")
    torch.cuda.synchronize()
    ctx.chunk_attn_paged(qq, case.k, case.v, case.table, case.lens_dev, case.indptr, out, lse,
                         scale=hd ** -0.5 if scale is None else scale, sliding_window=window, sink_tokens=sinks,
                         **_shape(case, q))
    if sync:
        ctx.sync()
        assert bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all())
    return out[:n], lse[:n]


def _check(ctx, case, q, *, window=0, sinks=0, tail=3):
    hd, keys = q.shape[2], max(case.lens)
    out, lse = _attend(ctx, case, q, window=window, sinks=sinks, tail=tail)
    want, z, amp = chunk_ref(case, q, scale=hd ** -0.5, window=window, sinks=sinks)
    vmax = max((float(v.abs().max()) for _, v in case.rows if v.numel()), default=1.0)
    assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, hd, keys, vmax)
    assert float((lse.double() - z).abs().max()) <= lse_tolerance(amp, hd, keys, float(z.abs().max()))
    return out, lse


SHAPES = [  # counts, lens, nkh, group, hd, page, window, sinks
    ([1], [1], 1, 8, 256, 64, 0, 0),
    ([1], [4000], 1, 8, 256, 64, 512, 4),
    ([5], [5], 1, 1, 64, 16, 0, 0),
    ([3, 0, 40, 1], [3, 7, 41, 300], 2, 4, 128, 16, 0, 0),
    ([130, 1, 17], [130, 260, 1000], 1, 8, 256, 64, 100, 3),
    ([33, 70], [500, 71], 1, 8, 512, 64, 0, 0),
    ([33, 70, 1], [500, 171, 900], 1, 4, 512, 16, 64, 5),
    ([64, 100], [64, 333], 4, 3, 128, 16, 0, 0),
    ([9, 20], [100, 77], 2, 5, 96, 48, 33, 1),
    ([50], [129], 1, 16, 64, 8, 0, 0),
    ([7, 12], [50, 12], 3, 1, 8, 1, 5, 2),
    ([40, 3], [99, 65], 1, 7, 200, 7, 0, 0),
    ([11], [400], 1, 8, 256, 200, 0, 0),
    ([300], [700], 1, 8, 256, 128, 1, 0),
    ([257], [900], 1, 1, 128, 64, 256, 300),
    ([2, 2, 2], [512, 513, 514], 1, 8, 384, 24, 512, 4),
    ([6], [200], 1, 24, 40, 16, 0, 0),
    # groups that do not fit into a CTA's rows, or into a tile's
    ([5, 1], [40, 300], 1, 130, 64, 16, 0, 0),
    ([3], [270], 1, 300, 128, 16, 20, 2),
    ([2, 1], [400, 77], 2, 40, 256, 64, 0, 0),
    ([4], [130], 1, 128, 512, 64, 100, 0),
]


@pytest.mark.parametrize("counts,lens,nkh,group,hd,page,window,sinks", SHAPES)
def test_chunk_attention(ctx, counts, lens, nkh, group, hd, page, window, sinks):
    case, q = _case(hd + sum(counts), counts, lens, nkh=nkh, group=group, hd=hd, page=page)
    _check(ctx, case, q, window=window, sinks=sinks)


FEW = [  # few query rows to a sequence: decode steps, some sequences idle, some with more tokens than the others
    ([1, 0, 1], [1, 40, 500], 1, 8, 256, 64, 0, 0),
    ([20, 0, 0], [333, 5, 9], 1, 1, 128, 16, 0, 0),
    ([5, 1, 0, 2], [70, 1, 3, 2], 2, 3, 96, 7, 0, 0),
    ([3, 1, 0], [120, 900, 4], 1, 4, 512, 16, 50, 5),
    ([7, 1], [200, 1000], 1, 2, 256, 64, 33, 3),
    ([1, 1], [17, 16], 4, 5, 64, 8, 0, 0),
    ([8], [8], 3, 1, 8, 1, 3, 1),
    ([1] * 9, [15 * i + 1 for i in range(9)], 1, 7, 200, 5, 0, 0),
    ([1, 2, 1, 0], [600, 601, 602, 3], 1, 3, 384, 24, 512, 4),
    ([6, 0], [300, 1], 1, 2, 320, 48, 100, 40),
    ([1], [3000], 2, 8, 512, 64, 2000, 200),
    ([1] * 60, [211 * i + 1 for i in range(60)], 1, 8, 512, 64, 0, 0),
    ([1] * 60, [211 * i + 1 for i in range(60)], 6, 2, 128, 16, 0, 0),  # more heads than a round of CTAs
    ([1] * 140, [(97 * i) % 2500 + 1 for i in range(140)], 1, 8, 256, 16, 600, 4),  # more sequences than a CTA deals out
]


@pytest.mark.parametrize("tail", [0, 3])  # (rows behind the last sequence count where the kernel is chosen)
@pytest.mark.parametrize("counts,lens,nkh,group,hd,page,window,sinks", FEW)
def test_chunk_attention_of_few_rows(ctx, counts, lens, nkh, group, hd, page, window, sinks, tail):
    case, q = _case(hd + sum(counts), counts, lens, nkh=nkh, group=group, hd=hd, page=page)
    _check(ctx, case, q, window=window, sinks=sinks, tail=tail)


@pytest.mark.parametrize("hd,group", [(64, 1), (256, 2), (512, 1), (512, 3)])
def test_values_that_are_not_finite_in_steps_of_few_rows(ctx, hd, group):
    counts, lens, window, sinks = [4, 1, 0, 0], [200, 40, 5, 9], 30, 3
    case, q = _case(hd, counts, lens, nkh=1, group=group, hd=hd, page=16)
    clean, lse0 = _attend(ctx, case, q, window=window, sinks=sinks)
    plant = [(0, 198, 5, float("inf")), (0, 199, hd - 1, float("nan")), (0, 1, 0, -float("inf")), (0, 168, 9, float("inf")),
             (0, 100, 4, float("nan")), (1, 39, 3, -float("inf"))]
    for b, r, d, x in plant:
        case.v[case.table_host[b, r // 16], r % 16, 0, d] = x
    out, lse = _attend(ctx, case, q, window=window, sinks=sinks)
    want = clean.double()
    for b, r, d, x in plant:
        for i in range(counts[b]):
            pos = lens[b] - counts[b] + i
            if r <= pos and (r > pos - window or r < sinks):
                want[case.indptr_host[b] + i, :, d] += x
    finite = want.isfinite()
    assert torch.equal(lse, lse0) and torch.equal(out.isfinite(), finite) and torch.equal(out[finite], clean[finite])
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want == float("inf"))


@pytest.mark.parametrize("hd", [128, 256, 512])
def test_steps_of_few_rows_out_of_the_ordinary(ctx, hd):
    """Single tokens (no rows behind them): scores that grow by thousands along the rows, missing pages, a key and a
    query that are not finite."""
    lens = [1500, 90]
    case, q = _case(hd, [1, 1], lens, nkh=1, group=8, hd=hd, page=16, spread=1.0)
    k, v = case.rows[0]
    k = (k * torch.linspace(0.02, 60.0, lens[0])[:, None, None]).half()
    case.rows[0] = (k, v)
    s = torch.arange(lens[0])
    case.k[case.table_host[0].long()[s // 16], s % 16] = k.cuda()
    _check(ctx, case, q, tail=0)
    clean, lse0 = _attend(ctx, case, q, tail=0)
    bad = q.clone()
    bad[0, 3, 1] = float("inf")
    page, row = int(case.table_host[1, 5]), 3
    was = case.k[page, row, 0, 2].clone()
    case.k[page, row, 0, 2] = float("nan")
    out, lse = _attend(ctx, case, bad, tail=0)
    assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all()) and bool(out[0, 3].isnan().all())
    others = torch.arange(8, device="cuda") != 3
    assert torch.equal(out[0, others], clean[0, others]) and torch.equal(lse[0, others], lse0[0, others])
    case.k[page, row, 0, 2] = was
    there = [torch.ones(n, dtype=torch.bool) for n in lens]
    for b, j, x in ((0, 2, -1), (0, 60, 1 << 30), (1, 0, case.k.shape[0])):
        case.table[b, j] = x
        there[b][j * 16:(j + 1) * 16] = False
    out, lse = _attend(ctx, case, q, tail=0, sync=False)
    with pytest.raises(G4AError, match="page id"):
        ctx.sync()
    want, z, amp = chunk_ref(case, q, scale=hd ** -0.5, there=there)
    vmax = max(float(v.abs().max()) for _, v in case.rows)
    assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, hd, 1500, vmax)
    assert float((lse.double() - z).abs().max()) <= lse_tolerance(amp, hd, 1500, float(z.abs().max()))


def test_sequences_whose_rows_overlap_are_refused_where_they_do_not_fit(ctx):
    """q_indptr that goes back and forth: each second sequence is in itself well formed, all together they are more than
    num_tokens; nothing is written out of bounds."""
    n, t = 40, 120
    case, q = _case(7, [t], [300], nkh=1, group=8, hd=128, page=16)
    table = case.table.expand(n, -1).contiguous()
    lens = torch.full((n,), 300, dtype=torch.int32, device="cuda")
    indptr = torch.tensor([0, t] * (n // 2) + [0], dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
    mass = torch.zeros((n, 1, 300), device="cuda")
    ctx.chunk_attn_paged(q, case.k, case.v, table, lens, indptr, out, lse, scale=0.1, **_shape(case, q))
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()
    ctx.paged_key_mass(q, lse, case.k, table, lens, indptr, mass, scale=0.1, **_shape(case, q))
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()


@pytest.mark.parametrize("hd,counts,lens,window,sinks", [
    (256, [1], [40_001], 0, 0), (512, [3], [30_000], 0, 0), (128, [20, 1], [9_000, 17_000], 0, 0),
    (256, [600], [5_003], 512, 4), (256, [900], [2_100], 0, 0), (512, [400], [3_300], 0, 0), (128, [1500], [1_900], 0, 0),
    (256, [1] * 40, [100 * i + 1 for i in range(40)], 0, 0), (512, [1] * 30, [333 * i + 9 for i in range(30)], 2000, 7)])
def test_chunk_attention_of_long_contexts(ctx, hd, counts, lens, window, sinks):
    """Tiles that are cut along the keys and joined, several tiles to a CTA."""
    case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=64)
    _check(ctx, case, q, window=window, sinks=sinks)


@pytest.mark.parametrize("seed", range(12))
def test_chunk_attention_of_drawn_shapes(ctx, seed):
    rnd = random.Random(seed)
    batch, nkh, hd = rnd.randint(1, 6), rnd.choice([1, 2, 4]), rnd.choice([16, 64, 96, 128, 176, 256, 256, 328, 512])
    counts = [rnd.choice([0, 1, rnd.randint(1, 20), rnd.randint(1, 200)]) for _ in range(batch)]
    lens = [max(1, t + rnd.choice([0, rnd.randint(0, 50), rnd.randint(0, 900)])) for t in counts]
    counts[0] = max(counts[0], 1)
    lens[0] = max(lens[0], counts[0])
    window = rnd.choice([0, 0, rnd.randint(1, 300)])
    case, q = _case(seed, counts, lens, nkh=nkh, group=rnd.choice([1, 2, 3, 8]), hd=hd, page=rnd.choice([1, 5, 8, 16, 40, 64]))
    _check(ctx, case, q, window=window, sinks=rnd.choice([0, 4, 130]) if window else 0)


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_values_that_are_not_finite_reach_only_the_tokens_that_see_them(ctx, hd):
    counts, lens, nkh, group = [60, 5], [200, 40], 2, 8
    case, q = _case(hd, counts, lens, nkh=nkh, group=group, hd=hd, page=16)
    window, sinks = 70, 3
    clean, lse0 = _attend(ctx, case, q, window=window, sinks=sinks)
    plant = [(0, 150, 0, 5, float("inf")), (0, 199, 1, 7, float("nan")), (0, 1, 1, 0, -float("inf")), (0, 75, 0, 9, float("inf")),
             (1, 37, 0, 3, float("nan")), (0, 100, 1, hd - 1, float("inf"))]
    for b, r, h, d, x in plant:
        case.v[case.table_host[b, r // 16], r % 16, h, d] = x
    out, lse = _attend(ctx, case, q, window=window, sinks=sinks)
    assert torch.equal(lse, lse0)
    want = clean.clone().double()
    for b, r, h, d, x in plant:
        for i in range(counts[b]):
            pos = lens[b] - counts[b] + i
            if r <= pos and (r > pos - window or r < sinks):
                want[case.indptr_host[b] + i, h * group:(h + 1) * group, d] += x
    finite = want.isfinite()
    assert torch.equal(out.isfinite(), finite)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want == float("inf"))
    # the other values come from the same weights and values
    assert torch.equal(out[finite], clean[finite])


@pytest.mark.parametrize("hd", [128, 256, 512])
def test_keys_and_queries_that_are_not_finite(ctx, hd):
    counts, lens = [40], [90]
    case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=16)
    clean, lse0 = _attend(ctx, case, q)
    r = 80  # seen by the tokens of rows 80 .. 89
    case.k[case.table_host[0, r // 16], r % 16, 0, 2] = float("nan")
    q = q.clone()
    q[4, 3, 1] = float("inf")
    out, lse = _attend(ctx, case, q)
    bad = torch.zeros(lse.shape, dtype=torch.bool, device="cuda")
    bad[30:] = True
    bad[4, 3] = True
    assert bool(out[bad].isnan().all()) and bool(lse[bad].isnan().all())
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], lse0[~bad])


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_scores_far_apart(ctx, hd):
    """Scores of thousands, growing along the rows: the running maximum is raised again and again."""
    counts, lens = [70], [1500]
    case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=16, spread=1.0)
    grow = torch.linspace(0.02, 60.0, lens[0])[:, None, None]
    k, v = case.rows[0]
    k = (k * grow).half()
    case.rows[0] = (k, v)
    s = torch.arange(lens[0])
    case.k[case.table_host[0].long()[s // 16], s % 16] = k.cuda()
    _check(ctx, case, q)
    case.rows[0] = ((-k).half(), v)
    case.k.neg_()
    _check(ctx, case, q, window=900, sinks=10)


def test_chunk_attention_skips_what_does_not_fit_and_reports_it(ctx):
    case, q = _case(3, [4, 6, 5], [50, 60, 20], nkh=1, group=8, hd=128, page=16)
    good, lse = _attend(ctx, case, q)
    case.lens_dev[1] = 3  # fewer rows than tokens
    out, got = _attend(ctx, case, q, sync=False)
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()
    assert bool((out[4:10] == 7.0).all()) and bool((got[4:10] == 7.0).all())
    assert torch.equal(out[:4], good[:4]) and torch.equal(out[10:], good[10:]) and torch.equal(got[10:], lse[10:])
    case.lens_dev[1] = 1 << 30
    out, _ = _attend(ctx, case, q, sync=False)
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()
    assert bool((out[4:10] == 7.0).all()) and torch.equal(out[10:], good[10:])


@pytest.mark.parametrize("hd", [128, 256, 512])
@pytest.mark.parametrize("page", [16, 5])
def test_rows_of_pages_that_are_not_there_are_not_seen(ctx, hd, page):
    case, q = _case(hd, [20, 3], [200, 90], nkh=1, group=8, hd=hd, page=page)
    there = [torch.ones(n, dtype=torch.bool) for n in case.lens]
    for b, j, bad in ((0, 2, -1), (0, 60 // page, 1 << 30), (1, 0, case.k.shape[0])):
        case.table[b, j] = bad
        there[b][j * page:(j + 1) * page] = False
    out, lse = _attend(ctx, case, q, sync=False)
    with pytest.raises(G4AError, match="page id"):
        ctx.sync()
    want, z, amp = chunk_ref(case, q, scale=hd ** -0.5, there=there)
    vmax = max(float(v.abs().max()) for _, v in case.rows)
    assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, hd, 200, vmax)
    assert float((lse.double() - z).abs().max()) <= lse_tolerance(amp, hd, 200, float(z.abs().max()))


# ------------------------------------------------------------------------------------------- key masses

def _mass(ctx, case, q, lse, mass, *, window=0, sinks=0, decay=1.0, sync=True):
    ctx.paged_key_mass(q, lse, case.k, case.table, case.lens_dev, case.indptr, mass, scale=q.shape[2] ** -0.5,
                       sliding_window=window, sink_tokens=sinks, decay=decay, **_shape(case, q))
    if sync:
        ctx.sync()
    return mass


def _check_mass(ctx, case, q, *, window=0, sinks=0, decay=1.0):
    hd = q.shape[2]
    _, z, amp = chunk_ref(case, q, scale=hd ** -0.5, window=window, sinks=sinks)
    lse = z.float()
    g = torch.Generator().manual_seed(9)
    before = torch.randn((len(case.lens), case.nkh, max(case.lens) + 5), generator=g).exp().cuda()
    for b, n in enumerate(case.lens):
        # new rows start from nothing, whatever was there; with decay 0 the others do too
        before[b, :, n - case.counts[b] if decay else 0:n] = float("nan")
    got = _mass(ctx, case, q, lse, before.clone(), window=window, sinks=sinks, decay=decay)
    want = mass_ref(case, q, lse, before, scale=hd ** -0.5, window=window, sinks=sinks, decay=decay)
    rows = max(case.counts) * q.shape[1] // case.nkh
    tol = mass_tolerance(amp, hd, rows, float(lse[lse.isfinite()].abs().max()))
    for b, n in enumerate(case.lens):
        assert torch.equal(got[b, :, n:], before[b, :, n:])
        assert bool(((got[b, :, :n].double() - want[b, :, :n]).abs() <= tol * want[b, :, :n] + 1e-37).all())
    return got


@pytest.mark.parametrize("decay", [1.0, 0.9, 0.0])
@pytest.mark.parametrize("counts,lens,nkh,group,hd,page,window,sinks", SHAPES + FEW)
def test_key_mass(ctx, counts, lens, nkh, group, hd, page, window, sinks, decay):
    case, q = _case(hd + sum(counts), counts, lens, nkh=nkh, group=group, hd=hd, page=page)
    _check_mass(ctx, case, q, window=window, sinks=sinks, decay=decay)


@pytest.mark.parametrize("hd,counts,lens,window,sinks", [
    (256, [1], [40_001], 0, 0), (512, [3], [30_000], 0, 0), (128, [20, 1], [9_000, 17_000], 0, 0),
    (256, [600], [5_003], 512, 4), (256, [900], [2_100], 0, 0), (512, [400], [3_300], 0, 0), (128, [1500], [1_900], 0, 0),
    (256, [1] * 40, [100 * i + 1 for i in range(40)], 0, 0)])
def test_key_mass_of_long_contexts(ctx, hd, counts, lens, window, sinks):
    case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=64)
    _check_mass(ctx, case, q, window=window, sinks=sinks)


def test_key_mass_of_rows_that_saw_nothing_and_of_missing_pages(ctx):
    case, q = _case(5, [6, 20], [30, 100], nkh=2, group=4, hd=128, page=16)
    _, z, _ = chunk_ref(case, q, scale=128 ** -0.5)
    lse = z.float()
    mass = torch.ones((2, 2, 100), device="cuda")
    want = _mass(ctx, case, q, lse, mass.clone())
    # a q row with an lse of -inf adds nothing: the rest is what the others add
    one = lse.clone()
    one[8, 3] = -float("inf")
    got = _mass(ctx, case, q, one, mass.clone())
    k = case.rows[1][0].cuda().double()[:83, 0]  # token 2 of sequence 1 has row 82
    w = torch.exp(q[8, 3].double() @ k.T * 128 ** -0.5 - z[8, 3])
    assert float(((want - got)[1, 0, :83].double() - w).abs().max()) <= 2.0 ** -18 * float(want.max())
    assert torch.equal(want[0], got[0]) and torch.equal(want[1, 1], got[1, 1])
    case.table[1, 2] = 1 << 20
    mass.fill_(3.0)
    got = _mass(ctx, case, q, lse, mass.clone(), sync=False)
    with pytest.raises(G4AError, match="page id"):
        ctx.sync()
    assert bool((got[1, :, 32:48] == 3.0).all())  # rows that are not there keep what they had
    assert torch.equal(got[1, :, :32], want[1, :, :32] + 2.0) or float((got[1, :, :32] - want[1, :, :32] - 2).abs().max()) < 1e-5
    assert float((got[1, :, 80:] - want[1, :, 80:]).abs().max()) == 0.0


def test_key_mass_skips_what_does_not_fit(ctx):
    case, q = _case(6, [4, 6], [50, 60], nkh=1, group=8, hd=128, page=16)
    lse = torch.zeros(q.shape[:2], device="cuda")
    mass = torch.full((2, 1, 55), 2.0, device="cuda")  # too few entries for the second sequence
    got = _mass(ctx, case, q, lse, mass, sync=False)
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()
    assert bool((got[1] == 2.0).all()) and not bool((got[0, 0, :50] == 2.0).any())


# --------------------------------------------------------------------------------------------- eviction

def _evict(ctx, case, mass, *, budget, sinks=0, recent=0, with_kept=True, sync=True):
    batch = len(case.lens)
    new = torch.full((batch,), -5, dtype=torch.int32, device="cuda")
    kept = torch.full((batch, case.nkh, budget), -7, dtype=torch.int32, device="cuda") if with_kept else None
    ctx.paged_kv_evict(case.k, case.v, case.table, case.lens_dev, mass, new, kept, budget=budget, sink_tokens=sinks,
                       recent_tokens=recent, num_kv_heads=case.nkh, head_dim=case.hd, page_size=case.page)
    if sync:
        ctx.sync()
    return new, kept


def _check_evict(ctx, case, mass, *, budget, sinks=0, recent=0, with_kept=True):
    k0, v0, m0 = case.k.clone(), case.v.clone(), mass.clone()
    want = evict_ref(mass.cpu(), case.lens, budget=budget, sinks=sinks, recent=recent)
    new, kept = _evict(ctx, case, mass, budget=budget, sinks=sinks, recent=recent, with_kept=with_kept)
    assert new.tolist() == [min(n, budget) for n in case.lens]
    if with_kept:
        assert torch.equal(kept.cpu(), want)
    for b, n in enumerate(case.lens):
        if n <= budget:
            continue
        i = torch.arange(budget)
        table = case.table_host[b].long()
        for h in range(case.nkh):
            j = want[b, h].long()
            to, at = (table[i // case.page], i % case.page, h), (table[j // case.page], j % case.page, h)
            k0[to], v0[to] = k0[at], v0[at]
            m0[b, h, :budget] = m0[b, h, j.cuda()]
    bits = lambda t: t.view(torch.int16 if t.dtype == torch.float16 else torch.int32)  # noqa: E731
    assert torch.equal(bits(case.k), bits(k0)) and torch.equal(bits(case.v), bits(v0))
    assert torch.equal(bits(mass), bits(m0))


EVICT = [  # lens, nkh, hd, page, budget, sinks, recent
    ([100], 1, 256, 16, 50, 4, 10),
    ([5, 1, 300, 0], 2, 128, 16, 5, 1, 2),
    ([1000, 999], 1, 512, 64, 999, 0, 0),
    ([2000, 50, 700], 4, 64, 8, 64, 4, 60),
    ([777], 3, 96, 7, 300, 0, 300),
    ([400], 1, 8, 1, 399, 399, 0),
    ([5000, 4097], 1, 256, 64, 2048, 4, 256),
    ([33000], 1, 128, 64, 9000, 4, 77),
    ([70001, 9], 2, 64, 48, 33333, 0, 5),
]


@pytest.mark.parametrize("lens,nkh,hd,page,budget,sinks,recent", EVICT)
@pytest.mark.parametrize("kind", ["spread", "ties", "rising", "falling", "odd"])
def test_evict(ctx, lens, nkh, hd, page, budget, sinks, recent, kind):
    case = Paged(sum(lens), lens, [0] * len(lens), nkh=nkh, hd=hd, page=page)
    top = max(lens) + 3
    g = torch.Generator().manual_seed(top)
    mass = torch.randn((len(lens), nkh, top), generator=g).exp()
    if kind == "ties":
        mass = (mass * 2).floor() / 2
    elif kind == "rising":
        mass = mass.sort(-1)[0]
    elif kind == "falling":
        mass = mass.sort(-1, descending=True)[0]
    elif kind == "odd":
        pick = torch.randint(0, 8, mass.shape, generator=g)
        for i, x in enumerate((float("nan"), 0.0, -0.0, float("inf"), -1.0, 1e-42)):
            mass[pick == i] = x
    mass = mass.cuda()
    _check_evict(ctx, case, mass, budget=budget, sinks=sinks, recent=recent, with_kept=kind != "rising")


def test_evict_reports_what_does_not_fit(ctx):
    case = Paged(4, [100, 100, 60], [0] * 3, nkh=1, hd=64, page=16)
    mass = torch.rand((3, 1, 100), device="cuda")
    case.lens_dev[1] = 101  # more rows than weights
    k0 = case.k.clone()
    new, kept = _evict(ctx, case, mass, budget=40, sync=False)
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()
    rows = lambda t, b: t[case.table_host[b].long()].view(torch.int16)  # noqa: E731
    assert new.tolist() == [40, 101, 40] and torch.equal(rows(case.k, 1), rows(k0, 1))
    case.lens_dev[1] = 100
    case.table[2, 1] = -1
    new, kept = _evict(ctx, case, mass, budget=40, sync=False)
    with pytest.raises(G4AError, match="page id"):
        ctx.sync()
    assert new.tolist() == [40, 40, 40]


# --------------------------------------------------------------------------------------------- together

def test_a_prompt_in_pieces_with_a_cache_kept_to_a_budget(ctx):
    """Append, attention, masses, eviction, chunk by chunk, then single tokens, against a cache of plain tensors."""
    nqh, nkh, hd, page, budget, sinks, recent = 8, 1, 256, 16, 150, 4, 40
    g = torch.Generator().manual_seed(2)
    batch, steps = 2, [(90, 100), (80, 33), (1, 70), (1, 1), (1, 1)]
    max_pages = 24
    table = torch.randperm(batch * max_pages, generator=g).int().view(batch, max_pages).cuda()
    kp = torch.full((batch * max_pages, page, nkh, hd), float("nan"), dtype=torch.float16, device="cuda")
    vp, mass = kp.clone(), torch.full((batch, nkh, page * max_pages), float("nan"), device="cuda")
    w = torch.ones(hd, dtype=torch.float16, device="cuda")
    lens, pos = [0] * batch, [0] * batch
    old = [torch.zeros((0, nkh), dtype=torch.float64, device="cuda")] * batch  # masses of the plain cache
    for counts in steps:
        n = sum(counts)
        raw = torch.randn((n, (nqh + 2 * nkh) * hd), generator=g).cuda()
        q, k, v = raw.split([nqh * hd, nkh * hd, nkh * hd], 1)
        seq = torch.tensor([b for b in range(batch) for _ in range(counts[b])], dtype=torch.int32, device="cuda")
        slot = torch.tensor([lens[b] + i for b in range(batch) for i in range(counts[b])], dtype=torch.int32, device="cuda")
        where = torch.tensor([pos[b] + i for b in range(batch) for i in range(counts[b])], dtype=torch.int32, device="cuda")
        cs = torch.zeros((n, hd), device="cuda")
        q16 = torch.zeros((n, nqh, hd), dtype=torch.float16, device="cuda")
        shape = dict(num_q_heads=nqh, num_kv_heads=nkh, head_dim=hd, page_size=page)
        ctx.rope_table(where, None, cs, head_dim=hd, theta=1e4)
        ctx.paged_qkv_prep(q, k, v, w, w, cs, q16, kp, vp, table, seq, slot, eps=1e-6, **shape)
        lens = [a + t for a, t in zip(lens, counts)]
        pos = [a + t for a, t in zip(pos, counts)]
        ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
        ip = torch.tensor([0, counts[0], n], dtype=torch.int32, device="cuda")
        out, lse = torch.zeros_like(q16), torch.zeros((n, nqh), device="cuda")
        ctx.chunk_attn_paged(q16, kp, vp, table, ld, ip, out, lse, scale=hd ** -0.5, **shape)
        ctx.paged_key_mass(q16, lse, kp, table, ld, ip, mass, scale=hd ** -0.5, **shape)
        ctx.sync()
        view = Paged.__new__(Paged)
        view.lens, view.counts, view.nkh, view.indptr_host = lens, list(counts), nkh, [0, counts[0], n]
        view.rows = []
        for b in range(batch):
            r = torch.arange(lens[b], device="cuda")
            at = (table[b].long()[r // page], r % page)
            view.rows.append((kp[at], vp[at]))
        want, z, amp = chunk_ref(view, q16, scale=hd ** -0.5)
        assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, hd, max(lens), float(max(v.abs().max() for _, v in view.rows)))
        before = torch.zeros((batch, nkh, page * max_pages), dtype=torch.float64, device="cuda")
        for b in range(batch):
            before[b, :, :len(old[b])] = old[b].T
        total = mass_ref(view, q16, lse, before, scale=hd ** -0.5)
        tol = 5 * mass_tolerance(amp, hd, max(counts) * nqh, float(z.abs().max()))  # five steps' sums
        for b in range(batch):
            assert bool(((mass[b, :, :lens[b]] - total[b, :, :lens[b]]).abs() <= tol * total[b, :, :lens[b]]).all())
        m = mass.clone()
        expect = evict_ref(m.cpu(), lens, budget=budget, sinks=sinks, recent=recent)
        new, kept = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros((batch, nkh, budget), dtype=torch.int32, device="cuda")
        ctx.paged_kv_evict(kp, vp, table, ld, mass, new, kept, budget=budget, sink_tokens=sinks, recent_tokens=recent,
                           num_kv_heads=nkh, head_dim=hd, page_size=page)
        ctx.sync()
        assert torch.equal(kept.cpu(), expect)
        lens = new.tolist()
        for b in range(batch):
            rows = kept[b, 0, :lens[b]].long()
            old[b] = total[b][:, rows].T
            r = torch.arange(lens[b], device="cuda")
            assert torch.equal(kp[table[b].long()[r // page], r % page], view.rows[b][0][rows])
            assert torch.equal(vp[table[b].long()[r // page], r % page], view.rows[b][1][rows])


@pytest.mark.parametrize("hd", [128, 256, 512])
def test_a_captured_step_follows_what_changes_between_replays(ctx, hd):
    """Attention, masses and eviction in one graph: lengths, pages and counts are read when it runs."""
    with g4attn.Context(0) as c:
        side = torch.cuda.Stream()
        c.set_stream(side.cuda_stream)
        counts, lens = [30, 1, 9], [300, 500, 9]
        case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=16)
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
        mass = torch.zeros((3, 1, case.table.shape[1] * 16), device="cuda")
        new = torch.zeros(3, dtype=torch.int32, device="cuda")

        def step():
            c.chunk_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, out, lse, scale=hd ** -0.5, **_shape(case, q))
            c.paged_key_mass(q, lse, case.k, case.table, case.lens_dev, case.indptr, mass, scale=hd ** -0.5, decay=0.0, **_shape(case, q))
            c.paged_kv_evict(case.k, case.v, case.table, case.lens_dev, mass, new, budget=200, sink_tokens=2, recent_tokens=20,
                             num_kv_heads=1, head_dim=hd, page_size=16)

        k0, v0 = case.k.clone(), case.v.clone()
        torch.cuda.synchronize()
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for counts2, lens2 in (([30, 1, 9], [300, 500, 9]), ([10, 29, 1], [250, 250, 5]), ([0, 40, 0], [3, 499, 9])):
            case.k.copy_(k0)
            case.v.copy_(v0)
            case.counts, case.lens = counts2, lens2
            case.indptr_host = [0, counts2[0], sum(counts2[:2]), sum(counts2)]
            case.lens_dev.copy_(torch.tensor(lens2, dtype=torch.int32))
            case.indptr.copy_(torch.tensor(case.indptr_host, dtype=torch.int32))
            rows = case.rows
            case.rows = []
            for b in range(3):
                r = torch.arange(lens2[b])
                at = (case.table_host[b].long()[r // 16], r % 16)
                case.rows.append((k0[at].cpu(), v0[at].cpu()))
            out.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.sync()
            n = sum(counts2)
            want, z, amp = chunk_ref(case, q, scale=hd ** -0.5)
            vmax = max(float(v.abs().max()) for _, v in case.rows)
            assert float((out[:n].double() - want[:n]).abs().max()) <= attn_tolerance(amp, hd, 500, vmax)
            assert bool((out[n:] == 7.0).all())
            assert new.tolist() == [min(x, 200) for x in lens2]
            for b, x in enumerate(lens2):  # every q row's weights sum to one; a sequence that was cut has lost some
                got = float(mass[b, 0, :min(x, 200)].double().sum())
                assert abs(got - 8 * counts2[b]) <= 1e-4 * 8 * counts2[b] if x <= 200 else got <= 8.001 * counts2[b]
            case.rows = rows
        del graph


@pytest.mark.parametrize("hd,counts,lens", [(256, [200, 3], [2000, 9000]), (512, [100, 1], [700, 20_000]), (128, [1] * 30, [900] * 30)])
def test_results_are_the_same_every_time(ctx, hd, counts, lens):
    case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=16)
    first, lse = _attend(ctx, case, q, window=700, sinks=4)
    mass = torch.rand((len(lens), 1, max(lens)), device="cuda")
    want = _mass(ctx, case, q, lse, mass.clone(), window=700, sinks=4)
    for _ in range(30):
        out, z = _attend(ctx, case, q, window=700, sinks=4)
        assert torch.equal(out, first) and torch.equal(z, lse)
        assert torch.equal(_mass(ctx, case, q, lse, mass.clone(), window=700, sinks=4), want)


def test_pools_beyond_32_bits_of_elements(ctx):
    """Pages whose elements lie beyond 2^32."""
    hd, page, nkh = 512, 64, 2
    pages = (1 << 32) // (hd * page * nkh) + 40
    case, q = _case(1, [30, 1], [400, 130], nkh=nkh, group=4, hd=hd, page=page)
    want, lse = _attend(ctx, case, q)
    mass = torch.rand((2, nkh, 400), device="cuda")
    total = _mass(ctx, case, q, lse, mass.clone())
    k, v = (torch.empty((pages, page, nkh, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    shift = pages - case.k.shape[0]
    k[shift:], v[shift:] = case.k, case.v
    small_k, small_v = case.k, case.v
    case.k, case.v, table = k, v, case.table
    case.table = table + shift
    out, z = _attend(ctx, case, q)
    assert torch.equal(out, want) and torch.equal(z, lse)
    got = _mass(ctx, case, q, lse, mass.clone())
    assert torch.equal(got, total)
    _evict(ctx, case, got, budget=100, sinks=3, recent=9)
    case.k, case.v, case.table = small_k, small_v, table
    _evict(ctx, case, total, budget=100, sinks=3, recent=9)
    bits = lambda t: t.view(torch.int16)  # noqa: E731
    assert torch.equal(got, total) and torch.equal(bits(k[shift:]), bits(small_k)) and torch.equal(bits(v[shift:]), bits(small_v))


@pytest.mark.parametrize("tokens", [1, 4])
def test_more_sequences_than_a_small_plan_holds(ctx, tokens):
    """More than 1,024 sequences (4 tokens of 4 heads each), and more than 128 of one token."""
    batch = 1100 if tokens > 1 else 150
    rnd = random.Random(tokens)
    counts = [rnd.choice([0, tokens, tokens]) for _ in range(batch)]
    lens = [max(1, c + rnd.randint(0, 60)) for c in counts]
    case, q = _case(3, counts, lens, nkh=1, group=8, hd=64, page=16)
    out, lse = _check(ctx, case, q, window=40, sinks=2)
    _check_mass(ctx, case, q, window=40, sinks=2, decay=0.5)


def test_many_tiles_in_one_call(ctx):
    """More tiles than a small plan holds, several heads, whole tiles and cut ones."""
    case, q = _case(4, [1500, 1300, 20, 900], [1500, 2000, 3500, 1000], nkh=4, group=48, hd=64, page=64)
    _check(ctx, case, q)
    _check_mass(ctx, case, q)


@pytest.mark.parametrize("hd", [128, 256, 512])
@pytest.mark.parametrize("scale", [-0.11, 0.0, 1.0])
def test_scales(ctx, hd, scale):
    """Scores that fall as the products rise, that are all alike, and that are not scaled; few rows and tiles of them."""
    for counts, lens in (([1, 1], [300, 40]), ([70], [200])):
        case, q = _case(hd, counts, lens, nkh=1, group=8, hd=hd, page=16, spread=0.5)
        out, lse = _attend(ctx, case, q, scale=scale)
        want, z, amp = chunk_ref(case, q, scale=scale)
        vmax = max(float(v.abs().max()) for _, v in case.rows)
        assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, hd, 300, vmax)
        assert float((lse.double() - z).abs().max()) <= lse_tolerance(amp, hd, 300, float(z.abs().max()))
        before = torch.zeros((len(lens), 1, max(lens)), device="cuda")
        got = before.clone()
        torch.cuda.synchronize()
        ctx.paged_key_mass(q, z.float(), case.k, case.table, case.lens_dev, case.indptr, got, scale=scale, **_shape(case, q))
        ctx.sync()
        want = mass_ref(case, q, z.float(), before, scale=scale)
        tol = mass_tolerance(amp, hd, max(counts) * 8, float(z.abs().max()))
        assert bool(((got.double() - want).abs() <= tol * want + 1e-37).all())


@pytest.mark.parametrize("counts,lens", [([1], [3000]), ([40], [90]), ([40], [30_000])])
def test_log_sum_exps_may_be_left_out(ctx, counts, lens):
    case, q = _case(1, counts, lens, nkh=1, group=8, hd=256, page=64)
    want, _ = _attend(ctx, case, q, tail=0)  # (rows behind the last sequence may choose the other kernel)
    out = torch.zeros_like(q)
    ctx.chunk_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, out, scale=256 ** -0.5, **_shape(case, q))
    ctx.sync()
    assert torch.equal(out, want)


def test_a_step_on_another_stream(ctx):
    """Calls on the context's stream follow each other there, whatever the current stream does."""
    with g4attn.Context(0) as c:
        side = torch.cuda.Stream()
        c.set_stream(side.cuda_stream)
        case, q = _case(11, [50, 1], [3000, 700], nkh=2, group=4, hd=256, page=16)
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
        mass = torch.zeros((2, 2, 3000), device="cuda")
        new = torch.zeros(2, dtype=torch.int32, device="cuda")
        want, z, amp = chunk_ref(case, q, scale=256 ** -0.5)
        torch.cuda.synchronize()
        shape = _shape(case, q)
        c.chunk_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, out, lse, scale=256 ** -0.5, **shape)
        c.paged_key_mass(q, lse, case.k, case.table, case.lens_dev, case.indptr, mass, scale=256 ** -0.5, **shape)
        got = mass_ref(case, q, z.float(), torch.zeros_like(mass), scale=256 ** -0.5)
        c.sync()
        assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, 256, 3000, max(float(v.abs().max()) for _, v in case.rows))
        for b, n in enumerate(case.lens):
            # (lse is the kernel's own here: twice its error)
            tol = mass_tolerance(amp, 256, 200, float(z.abs().max())) + 2 * lse_tolerance(amp, 256, 3000, float(z.abs().max()))
            assert bool(((mass[b, :, :n] - got[b, :, :n]).abs() <= tol * got[b, :, :n]).all())
        c.paged_kv_evict(case.k, case.v, case.table, case.lens_dev, mass, new, budget=500, recent_tokens=50, num_kv_heads=2,
                         head_dim=256, page_size=16)
        c.sync()
        assert new.tolist() == [500, 500]


def test_two_contexts_at_once(ctx):
    """Steps of two contexts on streams of their own, in flight together, give what each gives alone."""
    jobs = []
    for seed, hd, counts, lens in ((1, 128, [300, 1, 40], [2000, 900, 333]), (2, 512, [90], [5000]), (3, 256, [1] * 12, [800] * 12)):
        case, q = _case(seed, counts, lens, nkh=2, group=4, hd=hd, page=16)
        weights = torch.rand((len(lens), 2, max(lens)), generator=torch.Generator().manual_seed(seed)).cuda()
        jobs.append((case, q, weights))

    def step(c, case, q, weights):
        out, lse, mass = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda"), weights.clone()
        k, v, new = case.k.clone(), case.v.clone(), torch.zeros(len(case.lens), dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        shape = _shape(case, q)

        def run():
            c.chunk_attn_paged(q, k, v, case.table, case.lens_dev, case.indptr, out, lse, scale=0.1, **shape)
            c.paged_key_mass(q, lse, k, case.table, case.lens_dev, case.indptr, mass, scale=0.1, **shape)
            c.paged_kv_evict(k, v, case.table, case.lens_dev, mass, new, budget=200, recent_tokens=20, num_kv_heads=2,
                             head_dim=q.shape[2], page_size=16)
        return run, (out, lse, mass, k, v, new)

    with g4attn.Context(0) as a, g4attn.Context(0) as b:
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for c, s in zip((a, b), streams):
            c.set_stream(s.cuda_stream)
        for one in jobs:
            for other in jobs:
                alone = [step(ctx, *one), step(ctx, *other)]
                for run, _ in alone:
                    run()
                    ctx.sync()
                both = [step(a, *one), step(b, *other)]
                for run, _ in both:
                    run()
                a.sync()
                b.sync()
                for (_, want), (_, got) in zip(alone, both):
                    for x, y, name in zip(want, got, ("out", "lse", "mass", "k", "v", "new")):
                        kind = torch.int16 if x.dtype == torch.float16 else torch.int32  # (unused rows of the pools are NaN)
                        assert torch.equal(x.view(kind), y.view(kind)), name
