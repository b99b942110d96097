"""Steps that mix single tokens of many sequences with a piece of a prompt: in one call, and in two over slices of the same
tensors (the rows of q, of the page table and of the lengths), which is how to make them where the piece is long."""
import pytest
import torch

from chunk_ref import attn_tolerance, chunk_ref, lse_tolerance, mass_ref, mass_tolerance
from spec_ref import Paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("piece,group,hd,window,sinks", [
    (90, 1, 256, 0, 0), (40, 8, 256, 0, 0), (120, 4, 512, 300, 4), (33, 8, 128, 0, 0), (200, 2, 64, 90, 3)])
def test_single_tokens_and_a_piece_in_one_call_and_in_two(ctx, piece, group, hd, window, sinks):
    singles = 20
    counts, lens = [1] * singles + [piece], [70 * i + 1 for i in range(singles)] + [1500]
    case = Paged(piece, lens, counts, nkh=2, hd=hd, page=16)
    nqh = 2 * group
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((sum(counts), nqh, hd), generator=g) * 2).half().cuda()
    before = torch.randn((len(lens), 2, max(lens)), generator=g).exp().cuda()
    kw = dict(scale=hd ** -0.5, num_q_heads=nqh, num_kv_heads=2, head_dim=hd, page_size=16, sliding_window=window, sink_tokens=sinks)
    want, z, amp = chunk_ref(case, q, scale=hd ** -0.5, window=window, sinks=sinks)
    vmax = max(float(v.abs().max()) for _, v in case.rows)

    def calls(parts):
        out, lse, mass = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda"), before.clone()
        torch.cuda.synchronize()
        for b0, b1 in parts:
            i0, i1 = case.indptr_host[b0], case.indptr_host[b1]
            mine = (case.table[b0:b1], case.lens_dev[b0:b1], case.indptr[b0:b1 + 1] - i0)
            ctx.chunk_attn_paged(q[i0:i1], case.k, case.v, *mine, out[i0:i1], lse[i0:i1], **kw)
            ctx.paged_key_mass(q[i0:i1], lse[i0:i1], case.k, *mine, mass[b0:b1], decay=0.5, **kw)
        ctx.sync()
        return out, lse, mass

    for parts in ([(0, singles + 1)], [(0, singles), (singles, singles + 1)]):
        out, lse, mass = calls(parts)
        assert float((out.double() - want).abs().max()) <= attn_tolerance(amp, hd, 1500, vmax)
        assert float((lse.double() - z).abs().max()) <= lse_tolerance(amp, hd, 1500, float(z.abs().max()))
        total = mass_ref(case, q, lse, before, scale=hd ** -0.5, window=window, sinks=sinks, decay=0.5)
        tol = mass_tolerance(amp, hd, piece * group, float(z.abs().max()))
        for b, n in enumerate(lens):
            assert bool(((mass[b, :, :n] - total[b, :, :n]).abs() <= tol * total[b, :, :n] + 1e-37).all())
            assert torch.equal(mass[b, :, n:], before[b, :, n:])
