"""Tree attention with scores of any finite size."""
import pytest
import torch

from g4attn import G4AError
from spec_ref import Paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e2, 1e15, 1e28, 1e32])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_tree_attn_huge_scores_behind_rows_that_are_not_there(ctx, size, sign):
    """The first 128 keys lie on pages that are not there, so a row's first score of all comes late, as large or as
    low as it may be.  Two equal keys: the mean of their values."""
    hd, n, n_seq = 128, 130, 200  # (more sequences than CTAs, so that most do both stages of one; 32 rows fill a tile)
    case = Paged(1, [n] * n_seq, [1] * n_seq, nkh=1, hd=hd, page=64)
    case.table[:, :2] = -1
    last = case.table_host[:, 2].long()
    case.k[last, :2] = 0.5
    q = torch.full((n_seq, 32, hd), sign * size, device="cuda")
    out = torch.zeros_like(q)
    ctx.tree_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, None, out, num_q_heads=32,
                        num_kv_heads=1, head_dim=hd, page_size=64, max_tokens=1, scale=hd ** -0.5)
    with pytest.raises(G4AError, match="page id"):
        ctx.sync()
    v = torch.stack([r[1][128:, 0] for r in case.rows]).double()
    # two equal weights of 2^7: two terms of p, sums of four f32 numbers, one quotient
    tol = float(v.abs().max()) * 8 * 2.0 ** -23
    assert float((out.double().cpu() - v.mean(1)[:, None]).abs().max()) <= tol
