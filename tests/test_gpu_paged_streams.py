"""The paged attention's split rows on several streams of one captured graph."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16
from tests.test_gpu_paged import Cache, _dev, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


def test_two_streams_of_one_capture(ctx):  # noqa: F811
    """Calls on two streams that a capture forks, whose graph would run them beside each other: they share the workspace
    that split rows are joined in. Replayed with eager calls between."""
    import torch

    cs = [Cache(ctx, F16, 2, 128, 64, [6000, 5000], s) for s in (1, 2)]
    qs = [_dev(np.random.default_rng(s).standard_normal((2, 8 * 128)).astype(np.float32)) for s in (1, 2)]
    bs = [c.batch() for c in cs]
    want = [ctx.paged_attention(c.kv, c.pages, b, q, 8).clone() for c, b, q in zip(cs, bs, qs)]
    outs = [[torch.zeros_like(want[0]) for _ in range(4)] for _ in range(2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            main = torch.cuda.current_stream()
            side.wait_stream(main)
            for i in range(4):
                for j, s in enumerate((main, side)):
                    ctx.set_stream(s)
                    ctx.paged_attention(cs[j].kv, cs[j].pages, bs[j], qs[j], 8, out=outs[j][i])
            main.wait_stream(side)
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for _ in range(20):
        for o in outs[0] + outs[1]:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert all(torch.equal(o, want[j]) for o in outs[j])
            assert torch.equal(ctx.paged_attention(cs[j].kv, cs[j].pages, bs[j], qs[j], 8), want[j])
