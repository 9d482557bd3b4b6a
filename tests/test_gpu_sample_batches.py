"""kmoe_sample: a row's token is its own, whatever the batch; rows of many tokens that work-groups share, replayed in a
captured call with other values and settings, and on several streams."""
import numpy as np
import pytest

from tests.test_gpu_sample import _check, _dev, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


def test_a_rows_token_does_not_depend_on_the_number_of_rows(ctx):  # noqa: F811
    """600 tokens that fill no more than 600 groups of 64: work-groups share such a row up to 256 rows. The sum that top_p
    counts is right next to where one token more is kept: 31 chunks hold 410 times 2^-43 each in tokens of 0.4 of it."""
    import torch

    n = 70000
    x = np.full(n, -np.inf, np.float32)
    x[:38400:64] = -5000 * 2.0 ** -43
    x[0] = 0.0
    x[38 * 1024:] = -30.72
    x[38 * 1024::1024] = -30.316
    d = _dev(x)
    got = {}
    for S in (1, 2, 32, 256, 257, 300):
        rows, u, p = d.expand(S, n).contiguous(), torch.ones(S, device="cuda"), torch.full((S,), 0.5, device="cuda")
        got[S] = ctx.sample(rows, u, top_p=p).unique().tolist()
    assert len({tuple(v) for v in got.values()}) == 1 and len(got[1]) == 1, got
    assert got[1][0] in (299 * 64, 300 * 64)


N = 70001


def _rows(rng, kind):
    """A row of N logits, and settings under which it is greedy, gathered, shared, or nothing at all."""
    x = rng.standard_normal(N).astype(np.float32)
    if kind == "greedy":
        return x, 0.0, 0.9, 0.0
    if kind == "peaked":
        x[rng.integers(0, N, 20)] += np.float32(20)
        return x, 0.8, 0.95, 0.0
    if kind == "flat":
        return x, 1.3, 0.9, 0.0
    if kind == "equal":
        return np.round(x * 2) / 2, 1.0, 0.7, 0.0
    if kind == "min_p":
        return x, 1.0, 1.0, 0.01
    if kind == "both":
        return x, 2.0, 0.99, 0.02
    if kind == "whole":
        return x, 1.0, 1.0, 0.0
    return np.full(N, -np.inf, np.float32), 1.0, 0.9, 0.1


KINDS = ["greedy", "peaked", "flat", "equal", "min_p", "both", "whole", "nothing"]


@pytest.mark.parametrize("with_p,with_m", [(True, True), (True, False), (False, True)])
def test_captured_rows_that_are_shared_or_not(ctx, with_p, with_m):  # noqa: F811
    """Every row of every kind once, and each after every other: what a call leaves behind for the next one is nothing."""
    import torch

    rng = np.random.default_rng(11)
    S = 8
    x, u, t, p, m = (torch.zeros(s, device="cuda") for s in ((S, N), S, S, S, S))
    out = torch.zeros(S, dtype=torch.int32, device="cuda")
    how = dict(temperature=t, **({"top_p": p} if with_p else {}), **({"min_p": m} if with_m else {}))
    ctx.sample(x, u, out=out, **how)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.sample(x, u, out=out, **how)
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in range(10):
        kinds = [KINDS[(j * (1 + 2 * (i % 4)) + i) % len(KINDS)] for j in range(S)]
        hx, ht, hp, hm = (np.array(a, np.float32) for a in zip(*[_rows(rng, k) for k in kinds]))
        hu = rng.random(S).astype(np.float32)
        for d, h in ((x, hx), (u, hu), (t, ht), (p, hp), (m, hm)):
            d.copy_(_dev(h))
        g.replay()
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert np.array_equal(got, _check(ctx, hx, hu, temp=ht, p=hp if with_p else None, m=hm if with_m else None)), kinds
        g.replay()  # once more, after the eager call
        torch.cuda.synchronize()
        assert np.array_equal(got, out.cpu().numpy()), kinds


def test_streams_take_turns_with_shared_rows(ctx):  # noqa: F811
    """Calls of other rows and sizes on two streams of one context, one behind the other."""
    import torch

    rng = np.random.default_rng(12)
    calls = []
    for S in (2, 5, 40):
        rows = [_rows(rng, KINDS[1 + i % 5]) for i in range(S)]
        hx, ht, hp, hm = (np.array(a, np.float32) for a in zip(*rows))
        hu = rng.random(S).astype(np.float32)
        calls.append((dict(logits=_dev(hx), u=_dev(hu), temperature=_dev(ht), top_p=_dev(hp), min_p=_dev(hm)),
                      _check(ctx, hx, hu, temp=ht, p=hp, m=hm)))
    torch.cuda.synchronize()
    ss, outs = [torch.cuda.Stream() for _ in range(2)], []
    try:
        for i in range(24):
            ctx.set_stream(ss[i % 2])
            how, want = calls[i % 3]
            outs.append((ctx.sample(**how, out=torch.empty(len(want), dtype=torch.int32, device="cuda")), want))
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(torch.cuda.current_stream())
    assert all(np.array_equal(o.cpu().numpy(), w) for o, w in outs)
