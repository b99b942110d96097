"""Chunk attention's softmax weights: f16 for their product with V, with a place for the largest that leaves the small ones
their bits, whenever it is found.

Bound of one output, element by element.  With p_j the exact shares of the rows that are seen and A = sum p_j |v_j|:
 - a weight's exponent is off by the score's error (score_error, powers of two) and 2^-21 for exp2 and its argument, in the
   product and in the sum of the weights: 2 (ln 2 score_error + 2^-21) A;
 - its rounding to f16: 2^-11 of it, or 2^-25 below 2^-14.  The largest weight of every part of the keys is 2^3 at least, so 2^-25
   is 2^-28 of the largest share: 2^-11 A + 2^-28 max p_j sum |v_j|;
 - (keys / 16 + 36) additions of f32, cut off: 2^-23 A each;
 - the output's own rounding: 2^-11 of it, or 2^-25."""
import math

import pytest
import torch

from chunk_ref import chunk_ref, score_error, seen
from spec_ref import Paged

pytestmark = pytest.mark.gpu


def _bound(shares, v, out, amp, hd, keys):
    """shares [tokens, rows], v [rows, hd], out [tokens, hd] in f64."""
    dp = math.log(2) * score_error(amp, hd) + 2.0 ** -21
    a = shares @ v.abs()
    small = 2.0 ** -28 * shares.amax(1, keepdim=True) * ((shares > 0).double() @ v.abs())
    return (2 * dp + 2.0 ** -11 + (keys / 16 + 36) * 2.0 ** -23) * a + small + 2.0 ** -11 * out.abs() + 2.0 ** -25


@pytest.mark.parametrize("counts,lens,group,hd,window,sinks", [
    ([1, 1], [4000, 900], 8, 256, 0, 0), ([1] * 3, [5000, 70, 1], 4, 512, 600, 4), ([1] * 2, [3000, 2999], 8, 64, 0, 0),
    ([300], [2000], 8, 128, 0, 0), ([200, 3], [900, 5000], 8, 256, 512, 4), ([150], [1200], 4, 512, 0, 0)])
def test_every_output_within_what_the_roundings_allow(ctx, counts, lens, group, hd, window, sinks):
    case = Paged(sum(lens), lens, counts, nkh=1, hd=hd, page=16)
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn((sum(counts), group, hd), generator=g) * 3).half().cuda()
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    ctx.chunk_attn_paged(q, case.k, case.v, case.table, case.lens_dev, case.indptr, out, scale=hd ** -0.5,
                         sliding_window=window, sink_tokens=sinks, num_q_heads=group, num_kv_heads=1, head_dim=hd, page_size=16)
    ctx.sync()
    want, lse, amp = chunk_ref(case, q, scale=hd ** -0.5, window=window, sinks=sinks)
    for b, n in enumerate(lens):
        i0, t = case.indptr_host[b], counts[b]
        k, v = (x.cuda().double()[:, 0] for x in case.rows[b])
        see = seen(n, t, window, sinks)
        for h in range(group):
            x = q[i0:i0 + t, h].double() @ k.T * hd ** -0.5
            shares = torch.where(see, torch.exp(x - lse[i0:i0 + t, h, None]), 0.0)
            ref = want[i0:i0 + t, h]
            assert bool(((out[i0:i0 + t, h].double() - ref).abs() <= _bound(shares, v, ref, amp, hd, n)).all())


PAGE, HIGH, LONG = 64, 2, 131_000  # rows of a page; the page with the rows far above the others, in every sequence; rows


@pytest.mark.parametrize("below", [18, 19.4, 20, 21.45, 22, 24.2])
@pytest.mark.parametrize("hd,nkh,tokens", [(128, 2, 1), (256, 3, 1), (512, 3, 1), (128, 1, 40), (256, 1, 40), (512, 1, 20)])
def test_a_long_tail_behind_a_few_rows_far_above_it(ctx, hd, nkh, tokens, below):
    """Four rows `below` octaves above 131,000 others, behind the first 128 of these.  tokens > 1: tiles of query rows, as many as
    there are pairs of SMs and more, so that most of a row's keys are one thread's; one token: so many heads that a CTA has
    a quarter or half of a sequence's keys."""
    batch, group = 128, 8
    k = torch.zeros((2, PAGE, nkh, hd), dtype=torch.float16, device="cuda")
    v = torch.linspace(0.5, 2.0, hd, device="cuda").half().expand(2, PAGE, nkh, hd).contiguous()
    k[1, ::16, :, 0] = below * math.log(2)
    v[1, ::16] = 0.0
    table = torch.zeros((batch, -(-LONG // PAGE)), dtype=torch.int32, device="cuda")
    table[:, HIGH] = 1
    lens = torch.full((batch,), LONG, dtype=torch.int32, device="cuda")
    indptr = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * tokens
    q = torch.zeros((batch * tokens, nkh * group, hd), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
    torch.cuda.synchronize()
    ctx.chunk_attn_paged(q, k, v, table, lens, indptr, out, lse, scale=1.0, num_q_heads=nkh * group, num_kv_heads=nkh, head_dim=hd,
                         page_size=PAGE)
    ctx.sync()
    score = float(k[1, 0, 0, 0])
    tail = LONG - tokens + 1 + torch.arange(tokens, device="cuda").double() - 4  # rows of score 0 that a token sees
    z = tail + 4 * math.exp(score)
    want = (tail / z)[:, None] * v[0, 0, 0].double()
    amp = score * math.log2(math.e)
    dp = math.log(2) * score_error(amp, hd) + 2.0 ** -21
    small = 2.0 ** -28 * (math.exp(score) / z * tail)[:, None] * v[0, 0, 0].double()
    bound = (2 * dp + 2.0 ** -11 + (LONG / 16 + 36) * 2.0 ** -23 + 2.0 ** -11) * want + small + 2.0 ** -25
    got = out.view(batch, tokens, nkh * group, hd).double()
    assert bool(((got - want[:, None]).abs() <= bound[:, None]).all())
    assert float((lse.view(batch, tokens, -1).double() - z.log()[:, None]).abs().max()) <= \
        dp + (LONG / 16 + 36) * 2.0 ** -24 + 3 * float(z.log().max()) * 2.0 ** -24
