"""Heads of more than 256 dims: a tile's output goes through the place of its queries in shared memory, which the next tile's
queries are then copied to.  What a thread has stored or read there by ordinary instructions comes before a copy by TMA only
behind a proxy fence of that thread."""
import math
import re
from pathlib import Path

import pytest
import torch

from chunk_ref import score_error

SOURCE = Path(__file__).resolve().parent.parent / "gemma4-webgpu_b200" / "csrc" / "g4a_chunk_tc.cu"


def test_the_staging_place_is_handed_back_behind_a_proxy_fence():
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    last = text.index("mbar_arrive(staged)")
    used = text.rindex("smem + C::OFF_OUT", 0, last)
    between = text[used:last]
    fence, meet = between.find("if (!C::OWN_STAGING) fence_proxy_async_smem();"), between.rfind("__syncwarp();")
    assert 0 <= fence < meet, "every lane's fence, the warp's meeting, one lane's arrival"


@pytest.mark.gpu
@pytest.mark.parametrize("group,tokens,length,window", [(8, 5000, 5200, 60), (1, 30_000, 30_000, 20), (3, 6000, 6100, 60)])
def test_many_short_tiles_one_after_another(ctx, group, tokens, length, window):
    """Several whole tiles to a pair of CTAs, the next one's queries on their way while this one's output is written (by
    TMA where the group divides a CTA's rows); every element against the definition."""
    hd, page = 512, 64
    g = torch.Generator(device="cuda").manual_seed(group)
    k, v = (torch.randn((-(-length // page), page, 1, hd), generator=g, device="cuda").half() for _ in range(2))
    table = torch.arange(k.shape[0], dtype=torch.int32, device="cuda")[None]
    q = (torch.randn((tokens, group, hd), generator=g, device="cuda") * 2).half()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full_like(q, 7.0)
    call = lambda: ctx.chunk_attn_paged(q, k, v, table, ints(length), ints(0, tokens), out, scale=hd ** -0.5, sliding_window=window,  # noqa: E731
                                        num_q_heads=group, num_kv_heads=1, head_dim=hd, page_size=page)
    torch.cuda.synchronize()
    call()
    ctx.sync()
    first = out.clone()
    kk, vv = k.view(-1, hd), v.view(-1, hd)
    for t0 in range(0, tokens, 500):  # rows of the window alone
        n = min(500, tokens - t0)
        pos = length - tokens + t0 + torch.arange(n, device="cuda")
        r0 = max(0, int(pos[0]) - window + 1)
        row = torch.arange(r0, int(pos[-1]) + 1, device="cuda")
        see = (row <= pos[:, None]) & (row > pos[:, None] - window)
        x = torch.einsum("tgd,nd->tgn", q[t0:t0 + n].double(), kk[row].double()) * hd ** -0.5
        w = torch.softmax(x.masked_fill(~see[:, None], float("-inf")), -1)
        want, size = w @ vv[row].double(), w @ vv[row].double().abs()
        amp = float((q[t0:t0 + n].double().abs() @ kk[row].double().abs().T).max()) * hd ** -0.5 * math.log2(math.e)
        assert 2 * (math.log(2) * score_error(amp, hd) + 2.0 ** -21) + 40 * 2.0 ** -23 < 2.0 ** -11
        # weights in f16; their exponents and sums, as above; the output's rounding; the smallest weights
        assert bool(((first[t0:t0 + n].double() - want).abs() <= 2.0 ** -10 * size + 2.0 ** -11 * want.abs() + 2.0 ** -14).all())
    for _ in range(5):
        out.fill_(7.0)
        torch.cuda.synchronize()
        call()
        ctx.sync()
        assert torch.equal(out, first)
