"""Key masses of keys with infinite values: every query row's weight by its own score, whatever the row blocks are filled up
with where the heads of a group do not divide them."""
import pytest
import torch

from chunk_ref import chunk_ref, mass_ref, mass_tolerance
from spec_ref import Paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,group", [(100, 3), (90, 5), (30, 24), (2, 130), (60, 8), (3, 3)])
@pytest.mark.parametrize("hd", [128, 256, 512])
def test_keys_that_every_token_scores_minus_infinity(ctx, hd, count, group):
    length = 700
    case = Paged(hd + group, [length], [count], nkh=1, hd=hd, page=16)
    g = torch.Generator().manual_seed(group)
    q = (torch.randn((count, group, hd), generator=g) * 2).half()
    q[..., 5] = q[..., 5].abs() + 0.5
    q = q.cuda()
    rows = [0, 17, 300, length - count - 1]  # seen by all tokens
    k = case.rows[0][0]
    far = k.clone()
    far[rows, 0, 5] = -60_000.0  # (for the definition: as good as -inf, and finite)
    case.rows[0] = (far, case.rows[0][1])
    _, z, _ = chunk_ref(case, q, scale=hd ** -0.5)
    _, _, amp = chunk_ref(_with(case, k), q, scale=hd ** -0.5)
    at = torch.tensor(rows)
    case.k[case.table_host[0].long()[at // 16], at % 16, 0, 5] = -float("inf")
    before = torch.rand((1, 1, length), generator=g).cuda()
    mass, lse = before.clone(), z.float()
    torch.cuda.synchronize()
    ctx.paged_key_mass(q, lse, case.k, case.table, case.lens_dev, case.indptr, mass, num_q_heads=group, num_kv_heads=1, head_dim=hd,
                       page_size=16, scale=hd ** -0.5)
    ctx.sync()
    want = mass_ref(_with(case, far), q, lse, before, scale=hd ** -0.5)
    assert torch.equal(mass[0, 0, rows], before[0, 0, rows])
    tol = mass_tolerance(amp, hd, count * group, float(z.abs().max()))
    assert bool(((mass.double() - want).abs() <= tol * want + 1e-37).all())


def _with(case, k):
    case.rows[0] = (k, case.rows[0][1])
    return case
