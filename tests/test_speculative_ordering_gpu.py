"""What several warps of a speculative-step kernel hand to one another through shared memory.

Each case runs many times, behind other kernels and alone, so that warps come late in different places;
every result has to be the first one's to the bit, and the first is held to the 64-bit definition.
"""
import math
import random

import pytest
import torch

from g4attn import G4AError
from spec_ref import Paged, mask_tensor, tree_attn_ref, tree_masks, tree_tolerance

pytestmark = pytest.mark.gpu


def _tree(ctx, case, q, mask, out, window=0):
    nqh, hd = q.shape[1], q.shape[2]
    ctx.tree_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, mask, out, num_q_heads=nqh,
                        num_kv_heads=case.nkh, head_dim=hd, page_size=case.page, max_tokens=max(case.counts),
                        scale=hd ** -0.5, sliding_window=window, host_kv_lens=case.lens)


def _same_every_time(ctx, case, q, words, repeats=200, window=0):
    mask = mask_tensor(words)
    first = torch.zeros_like(q)
    _tree(ctx, case, q, mask, first, window)
    ctx.sync()
    ref, amp = tree_attn_ref(case, q, words, scale=q.shape[2] ** -0.5, window=window)
    vmax = max(float(v.double().abs().max()) for _, v in case.rows if v.numel())
    tol = tree_tolerance(amp, q.shape[2], max(case.lens), vmax, q.dtype == torch.float16)
    assert float((first.double().cpu() - ref).abs().max()) <= tol
    out = torch.zeros_like(q)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(repeats):
        out.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(1 + i % 3):
            _tree(ctx, case, q, mask, out, window)
        ctx.sync()
        differ += (out != first).any()
    assert int(differ) == 0


@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("batch,hd,group,most", [(33, 128, 3, 6), (70, 256, 8, 4), (140, 64, 2, 2)])
def test_tree_attn_of_33_to_512_sequences_is_the_same_every_time(ctx, fmt, batch, hd, group, most):
    """The table of sequences shares its place with the softmax weights: all warps are done with it before the
    first weight is written.  Short sequences, so that the first weights come early."""
    rnd = random.Random(batch)
    counts = [rnd.randint(1, most) for _ in range(batch)]
    lens = [c + rnd.randint(0, 90) for c in counts]
    case = Paged(batch, lens, counts, nkh=1, hd=hd, page=16)
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((sum(counts), group, hd), generator=g) * 2).to(fmt).cuda()
    _same_every_time(ctx, case, q, tree_masks(counts, rnd))


@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd,nkh,group,batch,most,longest", [
    (64, 4, 2, 60, 8, 300),   # 16 rows to a tile, several tiles of one or two stages to a CTA
    (256, 4, 8, 50, 8, 40),   # 64 rows, one stage to a tile
    (512, 2, 8, 100, 4, 150),
    (64, 1, 2, 512, 2, 90),   # as many sequences as the table holds
])
def test_tree_attn_of_several_tiles_to_a_cta_is_the_same_every_time(ctx, fmt, hd, nkh, group, batch, most, longest):
    """A tile's first maxima do not reach the sums of the tile before it."""
    rnd = random.Random(hd + batch)
    counts = [rnd.randint(1, most) for _ in range(batch)]
    lens = [c + rnd.randint(0, longest) for c in counts]
    case = Paged(batch, lens, counts, nkh=nkh, hd=hd, page=16)
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((sum(counts), nkh * group, hd), generator=g) * 2).to(fmt).cuda()
    _same_every_time(ctx, case, q, tree_masks(counts, rnd))


@pytest.mark.parametrize("hd,fmt", [(128, torch.float32), (256, torch.float16), (512, torch.float16)])
def test_tree_attn_with_missing_pages_is_the_same_every_time(ctx, hd, fmt):
    """Which rows of a stage are there, and what a tile's rows see, arrives with the stage: pages that are not there
    in every other stage, several stages to a CTA, another mask for each tile."""
    n_seq, group, t, n, page = 40, 4, 8, 1700, 16
    counts, lens = [t] * n_seq, [n] * n_seq
    case = Paged(hd, lens, counts, nkh=4, hd=hd, page=page)
    words = tree_masks(counts, random.Random(hd))
    gone = [[j for j in range((n - t) // page) if (j // 8 + b) % 2 == 0 and j % 3 == 0] for b in range(n_seq)]
    for b in range(n_seq):
        case.table[b, gone[b]] = -1
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((t * n_seq, 4 * group, hd), generator=g) * 2).to(fmt).cuda()
    mask = mask_tensor(words)
    first, out = torch.zeros_like(q), torch.zeros_like(q)

    def run(into):
        _tree(ctx, case, q, mask, into)
        with pytest.raises(G4AError, match="page id"):
            ctx.sync()

    run(first)
    vmax = max(float(v.double().abs().max()) for _, v in case.rows)
    worst = amp = 0.0
    for b in (0, 1, n_seq - 1):
        k, v = (x.double() for x in case.rows[b])
        keep = torch.tensor([r for r in range(n - t) if r // page not in set(gone[b])])
        for i in range(t):
            rows = torch.cat([keep, torch.tensor([n - t + j for j in range(t) if words[b * t + i] >> j & 1])])
            for h in range(0, 4 * group, 3):
                qq, kk = q[b * t + i, h].double().cpu(), k[rows, h // group]
                amp = max(amp, float((kk.abs() @ qq.abs()).max()) * hd ** -0.5 * math.log2(math.e))
                want = torch.softmax(kk @ qq * hd ** -0.5, 0) @ v[rows, h // group]
                worst = max(worst, float((first[b * t + i, h].double().cpu() - want).abs().max()))
    assert worst <= tree_tolerance(amp, hd, n, vmax, fmt == torch.float16)
    for _ in range(100):
        out.fill_(7.0)
        torch.cuda.synchronize()
        run(out)
        assert torch.equal(out, first)


@pytest.mark.parametrize("hd,fmt", [(128, torch.float32), (256, torch.float16)])
def test_tree_attn_of_non_finite_values_is_the_same_every_time(ctx, hd, fmt):
    """Infinite V values of drafted rows, in some tiles of a CTA and not in others: exactly the outputs of the tokens
    that attend to them are infinite, every time."""
    n_seq, group, t, nkh = 90, 4, 4, 4
    rnd = random.Random(hd)
    counts, lens = [t] * n_seq, [t + rnd.randint(0, 100) for _ in range(n_seq)]
    case = Paged(hd, lens, counts, nkh=nkh, hd=hd, page=16)
    words = tree_masks(counts, rnd, "star")  # token i sees the root and itself
    want = torch.zeros((n_seq * t, nkh * group, hd), dtype=torch.bool)
    for b in range(0, n_seq, 3):
        i, h, d = 1 + b % (t - 1), b % nkh, b % hd
        row = lens[b] - t + i
        case.v[case.table_host[b, row // 16], row % 16, h, d] = float("inf")
        want[b * t + i, h * group:(h + 1) * group, d] = True
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((n_seq * t, nkh * group, hd), generator=g) * 2).to(fmt).cuda()
    mask = mask_tensor(words)
    first, out = torch.zeros_like(q), torch.zeros_like(q)
    _tree(ctx, case, q, mask, first)
    ctx.sync()
    assert torch.equal(torch.isposinf(first).cpu(), want) and not bool(torch.isnan(first).any())
    for _ in range(100):
        out.fill_(7.0)
        torch.cuda.synchronize()
        _tree(ctx, case, q, mask, out)
        ctx.sync()
        assert torch.equal(out, first)


@pytest.mark.parametrize("fmt", [torch.float32, torch.float16])
@pytest.mark.parametrize("allowed", [0, 1, 5, 31])
@pytest.mark.parametrize("vocab", [20_011, 262_144, 600_001])
def test_top_k_of_equal_values_is_the_same_every_time(ctx, fmt, allowed, vocab):
    """Fewer values than are wanted above thousands of equal ones: the short lists of the join overflow, and its threads
    agree that they did.  Ties go to the lower id."""
    rows, k = 64, 32
    g = torch.Generator().manual_seed(vocab + allowed)
    x = torch.full((rows, vocab), -3.0, dtype=fmt)
    for r in range(rows):
        ids = torch.randperm(vocab, generator=g)[:allowed]
        x[r, ids] = torch.arange(allowed, dtype=fmt) * 0.25
        if r % 2:
            x[r][x[r] == -3.0] = -math.inf
    x = x.cuda()
    want = x.float().sort(dim=1, descending=True, stable=True)[1][:, :k].int().cpu()
    val = torch.zeros((rows, k), device="cuda")
    for _ in range(50):
        ids = torch.full((rows, k), -9, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        ctx.token_logprobs(x, None, None, None, val, ids)
        ctx.sync()
        assert torch.equal(ids.cpu(), want)
