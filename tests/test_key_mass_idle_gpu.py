"""Key masses of a step in which no sequence has new tokens: the call has room for tokens (a padded batch, a replayed graph),
so the weights fade as in any other step."""
import pytest
import torch

import g4attn
from g4attn import G4AError
from spec_ref import Paged

pytestmark = pytest.mark.gpu

IDLE = [  # tokens that q has room for, batch, rows of mass; 8 q heads
    (4, 3, 300),         # few rows to a sequence
    (40, 3, 300),        # tiles, one to a thread of the planning kernel
    (40, 3, 90_000),     # tiles, more than it has threads
    (4_500, 1_100, 70),  # more sequences than it has threads
]


def _idle(tokens, batch, room, *, hd, page=16):
    lens = [min(room, 300) * (b % 7) // 6 for b in range(batch)]
    lens[0] = min(room, 300)
    case = Paged(hd + batch, lens, [0] * batch, nkh=2, hd=hd, page=page)
    table = torch.zeros((batch, -(-room // page)), dtype=torch.int32, device="cuda")
    table[:, :case.table.shape[1]] = case.table
    case.table = table
    g = torch.Generator().manual_seed(batch)
    q = torch.randn((tokens, 8, hd), generator=g).half().cuda()
    mass = torch.randn((batch, 2, room), generator=g).exp().cuda()
    return case, q, torch.zeros((tokens, 8), device="cuda"), mass


def _call(c, case, q, lse, mass, **kw):
    c.paged_key_mass(q, lse, case.k, case.table, case.lens_dev, case.indptr, mass, num_q_heads=8, num_kv_heads=2,
                     head_dim=q.shape[2], page_size=case.page, scale=0.1, **kw)


def _faded(mass, lens, decay):
    want = mass.clone()
    for b, n in enumerate(lens):
        if n > 0:
            want[b, :, :n] = want[b, :, :n] * decay if decay else 0.0
    return want


@pytest.mark.parametrize("hd", [128, 256, 512])
@pytest.mark.parametrize("decay", [0.5, 0.0, 1.0])
@pytest.mark.parametrize("tokens,batch,room", IDLE)
def test_weights_fade_in_a_step_without_new_tokens(ctx, tokens, batch, room, decay, hd):
    case, q, lse, mass = _idle(tokens, batch, room, hd=hd)
    if decay == 0.0:
        mass[0, 0, 5] = float("nan")
    want = _faded(mass, case.lens, decay)
    torch.cuda.synchronize()
    _call(ctx, case, q, lse, mass, decay=decay, sliding_window=30, sink_tokens=2)
    ctx.sync()
    assert torch.equal(mass, want)


@pytest.mark.parametrize("tokens,batch,room", IDLE)
def test_a_sequence_that_does_not_fit_beside_idle_ones(ctx, tokens, batch, room):
    case, q, lse, mass = _idle(tokens, batch, room, hd=128)
    case.lens_dev[1] = room + 1
    want = _faded(mass, [n if b != 1 else 0 for b, n in enumerate(case.lens)], 0.5)
    torch.cuda.synchronize()
    _call(ctx, case, q, lse, mass, decay=0.5)
    with pytest.raises(G4AError, match="do not fit"):
        ctx.sync()
    assert torch.equal(mass, want)


def test_a_replayed_step_without_new_tokens():
    with g4attn.Context(0) as c:
        side = torch.cuda.Stream()
        c.set_stream(side.cuda_stream)
        case, q, lse, mass = _idle(40, 3, 300, hd=256)
        torch.cuda.synchronize()
        _call(c, case, q, lse, mass, decay=0.5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _call(c, case, q, lse, mass, decay=0.5)
        for counts in ([30, 0, 10], [0, 0, 0], [0, 20, 0], [0, 0, 0]):
            lens = [300, 200, 100]
            case.lens_dev.copy_(torch.tensor(lens, dtype=torch.int32))
            case.indptr.copy_(torch.tensor([0, counts[0], sum(counts[:2]), sum(counts)], dtype=torch.int32))
            case.k.nan_to_num_(0.0)
            before = mass.clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.sync()
            want = _faded(before, lens, 0.5)
            for b, t in enumerate(counts):
                if t == 0:
                    assert torch.equal(mass[b], want[b])
                else:
                    assert bool((mass[b, :, :lens[b] - t] > want[b, :, :lens[b] - t]).all())
        del graph
