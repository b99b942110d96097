"""A prompt longer than 64 tokens over the paged cache: appended whole, attended in chunks."""
import pytest
import torch

from spec_ref import Paged, tree_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,nqh,nkh,fmt,window", [(256, 8, 1, torch.float32, 0), (512, 8, 1, torch.float16, 0),
                                                   (128, 12, 4, torch.float16, 100), (64, 4, 2, torch.float32, 70)])
def test_a_long_prompt_in_chunks_of_64(ctx, hd, nqh, nkh, fmt, window):
    """Each chunk's kv_lens ends at the chunk: rows of later chunks, already in the pages, are not seen."""
    starts, n = [0, 37], [205, 130]  # cached rows before the prompt; tokens of the prompt
    lens = [a + b for a, b in zip(starts, n)]
    case = Paged(hd, lens, n, nkh=nkh, hd=hd, page=16)
    g = torch.Generator().manual_seed(hd)
    q = [torch.randn((t, nqh, hd), generator=g).to(fmt).cuda() for t in n]
    out = [torch.full_like(x, 5.0) for x in q]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for c in range(0, max(n), 64):
        t = [max(0, min(64, m - c)) for m in n]
        ends = [a + min(c + 64, m) for a, m in zip(starts, n)]
        qc = torch.cat([x[c:c + 64] for x in q])
        oc = torch.full_like(qc, 7.0)
        ctx.tree_attn_paged(qc, case.k, case.v, case.table, i32(ends), i32([0, t[0], t[0] + t[1]]), None, oc,
                            num_q_heads=nqh, num_kv_heads=nkh, head_dim=hd, page_size=16, max_tokens=64,
                            scale=hd ** -0.5, sliding_window=window, host_kv_lens=ends)
        ctx.sync()
        for x, y in zip(out, oc.split(t)):
            x[c:c + 64] = y
    group = nqh // nkh
    for b in range(2):
        k, v = (x.double() for x in case.rows[b])
        for h in range(0, nqh, 3):
            qq, kk, vv = q[b][:, h].double().cpu(), k[:, h // group], v[:, h // group]
            pos = starts[b] + torch.arange(n[b])[:, None]
            j = torch.arange(lens[b])[None]
            seen = (j <= pos) & ((j > pos - window) if window else True)
            s = torch.where(seen, qq @ kk.T * hd ** -0.5, -torch.inf)
            amp = float((qq.abs() @ kk.abs().T).max()) * hd ** -0.5 * 1.4427
            tol = tree_tolerance(amp, hd, lens[b], float(v.abs().max()), fmt == torch.float16)
            assert float((out[b][:, h].double().cpu() - torch.softmax(s, 1) @ vv).abs().max()) <= tol
