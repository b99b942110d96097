"""How a context's workspace grows: exactly and in place of the old one, until a call has been captured into a graph;
after that beside the old ones, which the graphs use."""
import pytest
import torch

import g4attn

pytestmark = pytest.mark.gpu
MB = 1 << 20


def _bytes(seqs, heads=64, hd=512):
    """What reserve_workspace(seqs, hd, heads) asks for, to the megabyte."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return (sms + seqs * heads + 1) * heads * (hd + 2) * 4


def _free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_growth_without_graphs_takes_what_is_asked_for(ctx):
    with g4attn.Context(0) as c:
        start = _free()
        for seqs in (8, 9, 10, 12):
            c.reserve_workspace(seqs, 512, 64)
            assert start - _free() <= _bytes(seqs) + 8 * MB  # the old one is gone, the new one no larger


def _captured(c):
    """A graph of a call that uses the workspace, and its output."""
    x = torch.randn((3, 5000), generator=torch.Generator().manual_seed(1)).cuda()
    tok, lp = torch.tensor([[1], [2], [3]], dtype=torch.int32, device="cuda"), torch.zeros((3, 1), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c.set_stream(side.cuda_stream)
    c.token_logprobs(x, tok, lp)
    torch.cuda.synchronize()
    want = lp.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.token_logprobs(x, tok, lp)
    return graph, lp, want, (x, tok, side)


def test_growth_keeps_what_graphs_use(ctx):
    with g4attn.Context(0) as c:
        graph, lp, want, keep = _captured(c)
        start = _free()
        for seqs in (8, 9, 18):
            c.reserve_workspace(seqs, 512, 64)
            lp.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(lp, want)
        assert start - _free() <= 2 * 2 * _bytes(9) + 16 * MB  # 9 doubled 8's; 18 fits in that or doubles it once
        del graph


def test_growth_beside_graphs_takes_less_where_double_does_not_fit(ctx):
    with g4attn.Context(0) as c:
        graph, lp, want, keep = _captured(c)
        c.reserve_workspace(64, 512, 64)
        torch.cuda.empty_cache()
        room = _bytes(70) + 256 * MB  # less than twice the present one
        assert room < 2 * _bytes(64)
        filler = torch.empty(_free() - room, dtype=torch.uint8, device="cuda")
        try:
            assert _free() <= room + 16 * MB
            c.reserve_workspace(70, 512, 64)
            with pytest.raises(g4attn.G4AError, match="workspace"):  # no room for that: refused, and the next call is sound
                c.reserve_workspace(700, 512, 64)
            lp.zero_()
            torch.cuda.synchronize()
            c.token_logprobs(keep[0], keep[1], lp)
            torch.cuda.synchronize()
            assert torch.equal(lp, want)
            lp.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(lp, want)
        finally:
            del filler
            torch.cuda.empty_cache()
        del graph
