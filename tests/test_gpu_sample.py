"""kmoe_sample (kmoe_sample.hip) against the definition in 64 bits: sizes from one
token on, equal logits, infinities and NaN, settings at their limits, rows that lie
apart, captured calls, refusals."""
import numpy as np
import pytest

from kestrel_amd.kmoe import KmoeError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from kestrel_amd.kmoe import Context

    c = Context(0)
    yield c
    c.close()


def _dev(a, dtype=np.float32):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def _reference(x, u, temp=1.0, k=0, p=1.0, m=0.0):
    """One row's token, its probability and the smallest distance of a decision from its border (relative)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return 0, 0.0
    if not temp > 0 or (not np.isnan(p) and p <= 0) or k == 1:
        return int(np.argmax(x)), 1.0
    if top == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore"):
            w = np.where(x == -np.inf, 0.0, np.exp((x - top) / temp))
        w[w < 2.0 ** -44] = 0.0  # the call's rule: weights are whole multiples of 2^-43, such a token is not drawn (u = 0)
    order = np.argsort(-x, kind="stable")
    if 0 < k < x.size:
        order = order[:k]
    if p < 1:
        run = np.cumsum(w[order])
        order = order[:int(np.searchsorted(run, float(p) * run[-1])) + 1]
    if m > 0:
        order = order[w[order] >= min(float(m), 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = 0.0 if not u > 0 else min(float(u), 1.0)
    i = int(np.searchsorted(run, u * run[-1], side="right"))
    if i == kept.size:  # u = 1: the last one of any weight
        i = int(np.flatnonzero(w[kept])[-1])
    return int(kept[i]), w[kept[i]] / run[-1]


def _check(ctx, x, u, temp=None, k=None, p=None, m=None, **kw):
    import torch

    S = x.shape[0]
    prob = torch.full((S,), float("nan"), device="cuda")
    arg = {n: None if v is None else _dev(np.broadcast_to(v, S), np.int32 if n == "top_k" else np.float32)
           for n, v in (("temperature", temp), ("top_k", k), ("top_p", p), ("min_p", m))}
    ids = ctx.sample(_dev(x), _dev(u), prob=prob, **arg, **kw)
    torch.cuda.synchronize()
    ids, prob = ids.cpu().numpy(), prob.cpu().numpy()
    row = lambda v, i, off: off if v is None else np.float32(np.broadcast_to(v, S)[i])  # noqa: E731
    for i in range(S):
        want, wp = _reference(x[i], np.float32(u[i]), row(temp, i, 1.0), int(row(k, i, 0)), row(p, i, 1.0), row(m, i, 0.0))
        assert ids[i] == want, (i, ids[i], want)
        # a weight and the sum are whole multiples of 2^-43 (half a unit each, and one for every token in the sum); the
        # probability is rounded to 32 bits once
        assert abs(prob[i] - wp) <= wp * (2.0 ** -23 + x.shape[1] * 2.0 ** -44) + 2.0 ** -43, (i, prob[i], wp)
    return ids


SETTINGS = [dict(), dict(temp=0.0), dict(k=1), dict(k=7), dict(p=0.9), dict(m=0.05), dict(temp=0.7, k=40, p=0.95),
            dict(temp=1.5, p=0.5, m=0.01), dict(temp=0.3, k=1000, p=0.99, m=0.001), dict(k=3, m=1.0), dict(temp=8.0, p=0.97)]


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 1000, 1024, 1025, 4095, 4097, 20011, 102403])
@pytest.mark.parametrize("how", range(len(SETTINGS)))
def test_matches_the_definition(ctx, n, how):
    rng = np.random.default_rng(100 * how + n)
    S = 3
    x = (rng.standard_normal((S, n)) * 3).astype(np.float32)
    x[0, rng.integers(0, n, 5)] += np.array([9, 8, 7, 6, 5], np.float32)  # a peaked row beside flat ones
    _check(ctx, x, rng.random(S).astype(np.float32), **SETTINGS[how])


def test_rows_with_settings_of_their_own(ctx):
    rng = np.random.default_rng(1)
    S, n = 300, 4000
    x = (rng.standard_normal((S, n)) * rng.choice([0.1, 1, 4], (S, 1))).astype(np.float32)
    _check(ctx, x, rng.random(S).astype(np.float32), temp=rng.choice([0, 0.1, 0.8, 1, 3], S), k=rng.choice([-1, 0, 1, 2, 50, 3999, 4000, 9999], S),
           p=rng.choice([0.0, 0.01, 0.4, 0.9, 1.0, 1.5, np.nan], S), m=rng.choice([-1, 0, 0.001, 0.2, 1.0, 2.0, np.nan], S))


@pytest.mark.parametrize("values", [1, 2, 5, 300])
@pytest.mark.parametrize("n", [5, 64, 1500, 50000])
def test_equal_logits_are_kept_by_index(ctx, values, n):
    """Few different values: every cut falls among equal ones. Borders of the draw and of top_p lie on sums exactly."""
    rng = np.random.default_rng(values * n)
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.999, 1.0], np.float32)
    x = rng.integers(0, values, (u.size, n)).astype(np.float32) / 4
    for how in (dict(), dict(k=3), dict(k=n // 2 + 1), dict(p=0.5), dict(p=0.75, k=max(2, n // 3)), dict(m=0.8)):
        _check(ctx, x if values > 1 else x * 0, u, **how)


def test_zeros_of_both_signs_are_equal(ctx):
    x = np.array([[-0.0, 0.0, -0.0, 0.0, -1.0]], np.float32)
    for u, want in ((0.0, 0), (0.4, 0), (0.5, 1), (0.9, 1)):
        assert _check(ctx, x, [u], k=2)[0] == want


def test_infinities_and_nan(ctx):
    inf, nan = np.inf, np.nan
    rows = [[nan, 1, 2, nan], [-inf, -inf, 0, -inf], [inf, 0, inf, 1], [nan, nan, nan, nan], [-inf, nan, -inf, -inf],
            [inf, nan, -inf, 3.0e38], [-3.0e38, 3.0e38, -inf, 3.0e38], [0, -3.0e38, 1.0e-40, -1.0e-40]]
    x = np.array(rows, np.float32)
    for u in (0.0, 0.3, 0.6, 0.99):
        for how in (dict(), dict(temp=0.0), dict(k=2), dict(p=0.6), dict(m=0.5), dict(temp=np.inf), dict(temp=np.nan),
                    dict(temp=1.0e-38), dict(temp=3.0e38, p=0.5)):
            _check(ctx, x, np.full(len(rows), u, np.float32), **how)


@pytest.mark.parametrize("u,want", [(-1.0, 0), (np.nan, 0), (0.0, 0), (1.0, 3), (7.0, 3), (np.inf, 3)])
def test_random_numbers_past_their_range(ctx, u, want):
    assert _check(ctx, np.zeros((1, 4), np.float32), [u])[0] == want


def test_a_temperature_that_makes_all_but_the_largest_vanish(ctx):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 3000)).astype(np.float32)
    for t in (1.0e-45, 1.0e-10, 1.0e-3):
        assert (_check(ctx, x, [0.0, 0.999], temp=t) == x.argmax(1)).all()


def test_every_token_is_drawn_as_often_as_it_weighs(ctx):
    """Evenly spaced u: a token's share of the draws is its probability, to two steps of u."""
    n, S = 50, 4096
    x = np.random.default_rng(6).standard_normal(n).astype(np.float32)
    ids = ctx.sample(_dev(np.broadcast_to(x, (S, n))), _dev((np.arange(S) + 0.5) / S)).cpu().numpy()
    w = np.exp(x.astype(np.float64))
    assert np.abs(np.bincount(ids, minlength=n) / S - w / w.sum()).max() <= 2 / S
    assert (np.diff(ids) >= 0).all()


def test_strided_rows_and_outputs(ctx):
    """Rows apart, at an address of 4 bytes; given outputs; positions advance; one row's result is its own."""
    import torch

    rng = np.random.default_rng(7)
    S, n = 9, 5003
    buf = torch.full((S * 6000 + 7,), float("nan"), device="cuda")
    x = buf[7:].view(S, 6000)[:, 1:1 + n]
    x.copy_(_dev(rng.standard_normal((S, n)) * 2))
    u, out, pos = _dev(rng.random(S)), torch.full((S,), -5, dtype=torch.int32, device="cuda"), _dev(np.arange(S), np.int32)
    p = _dev(np.full(S, 0.8))
    got = ctx.sample(x, u, top_p=p, out=out, pos_dev=pos, advance=3)
    assert got is out and pos.tolist() == list(range(3, 3 + S))
    _check(ctx, x.cpu().numpy(), u.cpu().numpy(), p=0.8)
    assert torch.equal(out, ctx.sample(x.contiguous(), u, top_p=p))
    for i in range(S):
        assert ctx.sample(x[i:i + 1], u[i:i + 1], top_p=p[i:i + 1]).item() == out[i].item()
    assert ctx.sample(x[:0], u[:0]).numel() == 0


def test_a_captured_call_reads_what_the_arrays_hold(ctx):
    import torch

    rng = np.random.default_rng(8)
    S, n = 5, 30000
    x, u, t = torch.empty((S, n), device="cuda"), torch.empty(S, device="cuda"), torch.empty(S, device="cuda")
    k, out = torch.empty(S, dtype=torch.int32, device="cuda"), torch.empty(S, dtype=torch.int32, device="cuda")
    for a in (x, u, t, k):
        a.zero_()
    ctx.sample(x, u, temperature=t, top_k=k, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.sample(x, u, temperature=t, top_k=k, out=out)
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in range(6):
        hx, hu = (rng.standard_normal((S, n)) * (1 + i)).astype(np.float32), rng.random(S).astype(np.float32)
        ht, hk = np.float32(rng.choice([0, 0.5, 1.3], S)), rng.choice([0, 5, 2000], S)
        for d, h in ((x, hx), (u, hu), (t, ht), (k, hk)):
            d.copy_(_dev(h, np.int32 if d is k else np.float32))
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), _check(ctx, hx, hu, temp=ht, k=hk))


def test_two_streams(ctx):
    """Calls on other streams than the last one's."""
    import torch

    rng = np.random.default_rng(9)
    x, u = _dev(rng.standard_normal((4, 60000))), _dev(rng.random(4))
    want = ctx.sample(x, u).clone()
    torch.cuda.synchronize()
    ss, outs = [torch.cuda.Stream() for _ in range(2)], []
    try:
        for i in range(20):
            ctx.set_stream(ss[i % 2])
            outs.append(ctx.sample(x, u, out=torch.empty_like(want)))
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(torch.cuda.current_stream())
    assert all(torch.equal(o, want) for o in outs)


def test_refusals(ctx):
    import torch

    x, u = torch.zeros((4, 100), device="cuda"), torch.zeros(4, device="cuda")
    bad = [dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.t()), dict(u=u[:3]), dict(u=u.double()),
           dict(temperature=u.half()), dict(top_k=u), dict(top_p=u[:1]), dict(min_p=u.cpu()), dict(out=u), dict(prob=u.double()),
           dict(pos_dev=torch.zeros(4, dtype=torch.int64, device="cuda")), dict(u=torch.zeros((4, 2), device="cuda")[:, 0])]
    for b in bad:
        with pytest.raises(ValueError):
            ctx.sample(**{**dict(logits=x, u=u), **b})
    buf = torch.zeros(500, device="cuda")
    i32 = buf.view(torch.int32)
    for b in (dict(logits=buf[:400].view(4, 100), out=i32[398:402]), dict(prob=u), dict(prob=buf[:4], out=i32[3:7]),
              dict(pos_dev=i32[:4], out=i32[:4]), dict(top_p=buf[4:8], prob=buf[7:11])):
        with pytest.raises(KmoeError) as e:
            ctx.sample(**{**dict(logits=x, u=u), **b})
        assert e.value.status == -1
    # between two rows nothing is overlapped
    ctx.sample(buf[:480].view(4, 120)[:, :100], u, out=i32[100:104], prob=buf[224:228])
    f = ctx.lib.kmoe_sample
    o = torch.zeros(8, dtype=torch.int32, device="cuda")
    for rows, n, stride in ((4, 0, 0), (4, -1, 5), (4, (1 << 20) + 1, 1 << 21), (-1, 100, 100), (4, 100, 99), ((1 << 20) + 1, 1, 1), (2, 100, 2 ** 62)):
        assert f(ctx.h, x.data_ptr(), rows, n, stride, None, u.data_ptr(), o.data_ptr(), None, None, 0) == -1, (rows, n, stride)
    for args in ((0, u.data_ptr(), o.data_ptr()), (x.data_ptr(), 0, o.data_ptr()), (x.data_ptr(), u.data_ptr(), 0)):
        assert f(ctx.h, args[0], 4, 100, 100, None, args[1], args[2], None, None, 0) == -1
    assert f(None, x.data_ptr(), 4, 100, 100, None, u.data_ptr(), o.data_ptr(), None, None, 0) == -1
    assert f(ctx.h, 0, 0, 100, 100, None, 0, 0, None, None, 0) == 0
    assert f(ctx.h, x.data_ptr(), 4, 100, 100, None, u.data_ptr(), o.data_ptr(), None, None, 0) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", [8191, 8193, 12289, 1 << 20])
def test_the_last_token_of_long_rows(ctx, n):
    """The largest logit, the k-th and the drawn one at the ends of chunks and rows."""
    rng = np.random.default_rng(n)
    at = sorted({i for i in (0, 63, 64, 4095, 4096, 8191, n - 2, n - 1) if i < n})
    x = rng.standard_normal((len(at), n)).astype(np.float32)
    x[np.arange(len(at)), at] = 30.0
    for how in (dict(temp=0.0), dict(k=5), dict(), dict(p=0.9)):
        assert (_check(ctx, x, np.full(len(at), 0.5, np.float32), **how) == at).all()
    x[:, n - 64:] = 40.0  # a whole group of equal ones at the end
    for how in (dict(k=5), dict(p=0.5), dict(m=0.9), dict()):
        _check(ctx, x[:2], [0.1, 0.99], **how)


@pytest.mark.parametrize("how", [dict(k=900), dict(k=5000), dict(p=0.9999), dict(m=1e-6), dict(temp=1.3, p=0.9), dict(temp=50.0, k=3000, p=0.7, m=0.9)])
def test_more_tokens_kept_than_fit_the_candidates(ctx, how):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((4, 60001)) * np.array([[0.01], [0.5], [2], [6]])).astype(np.float32)
    _check(ctx, x, np.array([0.001, 0.3, 0.9, 0.9999], np.float32), **how)


def test_more_rows_than_the_workspace_holds(ctx):
    """The rows go by parts then: 16 MB hold 17476 rows of 9 chunks."""
    import torch

    S, n = 20900, 8200
    x = torch.randn((S, n), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    u = torch.rand(S, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    k = torch.full((S,), 30, dtype=torch.int32, device="cuda")
    got = ctx.sample(x, u, top_k=k)
    for i in list(range(17470, 17485)) + [0, S - 1]:
        assert got[i].item() == _reference(x[i].cpu().numpy(), u[i].item(), k=30)[0]


@pytest.mark.parametrize("S", [1, 3, 17, 40, 200, 256, 257])
def test_rows_that_work_groups_share(ctx, S):
    """Rows of which much is kept beside others, at every number of work-groups that share one."""
    rng = np.random.default_rng(S)
    n = 70001
    x = (rng.standard_normal((S, n)) * rng.choice([0.3, 1, 2, 5], (S, 1))).astype(np.float32)
    x[::3, 7] += 25.0  # (and rows that are not flat)
    x[1::5] = np.round(x[1::5] * 4) / 4  # equal logits at every cut
    x[2::7, ::2] = -np.inf
    for how in (dict(p=rng.choice([0.3, 0.9, 0.999], S), temp=rng.choice([0.7, 1.0, 2.0], S)), dict(m=rng.choice([0.0, 1e-4, 0.01], S), temp=1.5),
                dict(p=rng.choice([0.6, 0.95, 1.0], S), m=rng.choice([0.0, 1e-3, 0.05], S), k=rng.choice([0, 0, 20, 5000], S))):
        _check(ctx, x, rng.random(S).astype(np.float32), **how)
