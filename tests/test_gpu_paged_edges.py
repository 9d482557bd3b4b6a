"""The paged cache's entry points at their edges: as many sequences as a call
takes, windows past 32 bits, tables without columns, odd addresses, lengths and
row starts that make no sense, captured prompt chunks, two captured graphs."""
from types import SimpleNamespace

import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0
from tests.test_gpu_paged import TYPES, Cache, _attend, _close, _dev, _reference, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,most", [(4, 2, 64, 1), (4, 2, 128, 1), (16, 1, 64, 3), (16, 1, 128, 3)])
def test_as_many_sequences_as_a_call_takes(ctx, t, nh, nkv, hd, most):  # noqa: F811
    rng = np.random.default_rng(hd)
    lens = rng.integers(most, 70, 4096).tolist()
    rows = None if most == 1 else rng.integers(1, most + 1, 4096).tolist()
    c = Cache(ctx, t, nkv, hd, 32, lens, 1)
    S = 4096 if rows is None else sum(rows)
    q = rng.standard_normal((S, nh, hd)).astype(np.float32)
    got = _attend(c, q, nh, rows).reshape(S, nh, hd)
    assert np.isfinite(got).all()
    pick = [0, 1, 255, 256, 257, 2048, 4094, 4095] + rng.integers(0, 4096, 40).tolist()
    rs = np.concatenate([[0], np.cumsum([1] * 4096 if rows is None else rows)])
    at = np.concatenate([np.arange(rs[b], rs[b + 1]) for b in pick])
    sub = SimpleNamespace(kv=c.kv, lens=[lens[b] for b in pick], hk=[c.hk[b] for b in pick], hv=[c.hv[b] for b in pick])
    ref, tol, _ = _reference(sub, q[at], None if rows is None else [rows[b] for b in pick], nh)
    _close(got[at], ref, tol)


@pytest.mark.parametrize("rows", [None, [1, 40]])
def test_windows_past_32_bits(ctx, rows):  # noqa: F811
    nh, nkv, hd = 8, 2, 64
    c = Cache(ctx, F16, nkv, hd, 32, [70, 90], 3)
    q = np.random.default_rng(3).standard_normal((2 if rows is None else 41, nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, rows, nh)
    for window, sink in ((0, 0), (2 ** 31 - 1, 0), (2 ** 31, 5), (2 ** 40, 0), (2 ** 62, 2 ** 62), (1, 2 ** 31 - 1), (1, 2 ** 31),
                         (7, 2 ** 62)):
        _close(_attend(c, q, nh, rows, window=window, n_sink=sink), ref, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,rows", [(4, None), (16, [3])])
def test_lengths_past_the_table(ctx, t, nh, rows):  # noqa: F811
    """Rows near position 2^31 of a table of 96 positions: they see those that the window leaves."""
    nkv, hd = 1, 64
    c = Cache(ctx, t, nkv, hd, 32, [96], 11)
    S = 1 if rows is None else rows[0]
    q = np.random.default_rng(11).standard_normal((S, nh, hd)).astype(np.float32)
    b = c.batch(rows, lens=[2 ** 31 - 1])
    for window, sink, n in ((0, 0, 96), (50, 0, 0), (50, 5, 5), (2 ** 31 - 96, 0, None), (2 ** 40, 0, 96)):
        out = ctx.paged_attention(c.kv, c.pages, b, _dev(q.reshape(S, -1)), nh, window=window, n_sink=sink)
        for i in range(S):
            at = 2 ** 31 - 1 - S + i  # the row's position
            p = np.arange(96)
            see = p < n if n is not None else p > at - window
            sub = SimpleNamespace(kv=c.kv, lens=[int(see.sum())], hk=[c.hk[0][see]], hv=[c.hv[0][see]])
            ref, tol, _ = _reference(sub, q[i:i + 1], None, nh)
            _close(out[i:i + 1].cpu().numpy(), ref, tol)


@pytest.mark.parametrize("t", TYPES)
def test_a_table_without_columns(ctx, t):  # noqa: F811
    import torch

    nh, nkv, hd = 4, 2, 128
    c = Cache(ctx, t, nkv, hd, 64, [5, 70], 4)
    b = ctx.paged_batch(torch.empty((2, 0), dtype=torch.int32, device="cuda"), _dev([5, 70], np.int32))
    keep = c.pages.clone()
    q = torch.ones((2, nh * hd), device="cuda")
    kv = torch.ones((2, nkv * hd), device="cuda")
    out = ctx.paged_attention(c.kv, c.pages, b, q, nh, out=torch.full_like(q, 7.0))
    ctx.paged_kv_store(c.kv, c.pages, b, kv, kv)
    back = ctx.paged_kv_read(c.kv, c.pages, b)
    torch.cuda.synchronize()
    assert not out.any() and not back[0].any() and not back[1].any() and torch.equal(keep, c.pages)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_at_odd_addresses(ctx, t, hd):  # noqa: F811
    """q, k, v and the outputs four bytes past a multiple of 16."""
    import torch

    nh, nkv, lens = 6, 2, [33, 1, 64]
    c = Cache(ctx, t, nkv, hd, 32, lens, 5)
    d = Cache(ctx, t, nkv, hd, 32, lens, 5)
    rs = np.concatenate([[0], np.cumsum(lens)])
    S = int(rs[-1])

    def odd(x):
        y = torch.zeros(x.size + 1, device="cuda")[1:].view(x.shape[0], -1)
        y.copy_(_dev(x.reshape(x.shape[0], -1)))
        assert y.data_ptr() % 16 == 4
        return y

    d.pages.fill_(0xff)
    ctx.paged_kv_store(d.kv, d.pages, d.batch(lens), odd(np.concatenate(c.k)), odd(np.concatenate(c.v)))
    assert torch.equal(c.pages, d.pages)
    q = np.random.default_rng(5).standard_normal((S, nh, hd)).astype(np.float32)
    out, rot = (odd(np.zeros((S, nh * hd), np.float32)) for _ in range(2))
    a = ctx.paged_attention(c.kv, c.pages, c.batch(lens), _dev(q.reshape(S, -1)), nh)
    ctx.paged_attention(c.kv, c.pages, c.batch(lens), odd(q), nh, out=out)
    assert torch.equal(a, out)
    inv = _dev((10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)).astype(np.float32))
    args = odd(q), odd(np.concatenate(c.k)), odd(np.concatenate(c.v)), nh, hd, inv, True
    a = ctx.paged_rope_kv_store(c.kv, c.pages, c.batch(lens), *(x.clone() for x in args[:3]), *args[3:])
    ctx.paged_rope_kv_store(d.kv, d.pages, d.batch(lens), *args, q_out=rot)
    assert torch.equal(a, rot) and torch.equal(c.pages, d.pages)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh", [2, 16])
def test_lengths_and_row_starts_that_make_no_sense(ctx, t, nh):  # noqa: F811
    """Nothing outside the call's rows is written; rows that one sequence alone has are right, and those of a sequence
    that is shorter than they are many see nothing."""
    import torch

    nkv, hd, lens = 1, 64, [50, 60, 70, 80, 40]
    c = Cache(ctx, t, nkv, hd, 32, lens, 6)
    rs = _dev([5, 2, 9, -4, 3, 100], np.int32)  # rows none, 2 .. 7, none, 0 .. 2, 3 .. 7
    q = np.random.default_rng(6).standard_normal((8, nh, hd)).astype(np.float32)
    b = ctx.paged_batch(_dev(c.table), _dev(lens, np.int32), rs, 8)
    out = torch.full((10, nh * hd), 3.0, device="cuda")
    ctx.paged_attention(c.kv, c.pages, b, _dev(q.reshape(8, -1)), nh, out=out[:8])
    sub = SimpleNamespace(kv=c.kv, lens=[80], hk=[c.hk[3]], hv=[c.hv[3]])
    ref, tol, _ = _reference(sub, q[:3], [3], nh)
    got = out.cpu().numpy()
    _close(got[:2], ref[:2], tol[:2])
    assert (got[8:] == 3.0).all()
    kv = torch.ones((10, nkv * hd), device="cuda")
    ctx.paged_kv_store(c.kv, c.pages, b, kv[:8], kv[:8])
    ctx.paged_kv_read(c.kv, c.pages, b)
    torch.cuda.synchronize()
    low = [-2 ** 31, -1, 0, 3, 2]
    for rows in (None, [1, 1, 2, 2, 30]):
        q = np.random.default_rng(7).standard_normal((5 if rows is None else 36, nh, hd)).astype(np.float32)
        n = [0, 0, 0, 3, 2]
        sub = SimpleNamespace(kv=c.kv, lens=n, hk=[x[:m] for x, m in zip(c.hk, n)], hv=[x[:m] for x, m in zip(c.hv, n)])
        c2 = Cache(ctx, t, nkv, hd, 32, n, 8)
        sub.hk, sub.hv = c2.hk, c2.hv
        ref, tol, S = _reference(sub, q, rows, nh)
        out = ctx.paged_attention(c2.kv, c2.pages, c2.batch(rows, lens=low), _dev(q.reshape(S, -1)), nh)
        _close(out.cpu().numpy(), ref, tol)


@pytest.mark.parametrize("t", TYPES)
def test_captured_chunks_follow_their_rows(ctx, t):  # noqa: F811
    """Store, read-back and attention of up to 130 rows captured once and replayed with other row counts and lengths;
    eager calls between the replays give the same bits. Rows behind the last sequence stay as they were."""
    import torch

    nh, nkv, hd, S = 16, 4, 128, 130
    c = Cache(ctx, t, nkv, hd, 64, [700, 300, 900], 9)
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v = (torch.zeros((S, w), device="cuda") for w in (nh * hd, nkv * hd, nkv * hd))
    qr, o = torch.zeros_like(q), torch.zeros_like(q)
    lens, rs = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    b = ctx.paged_batch(_dev(c.table), lens, rs, S)
    inv = _dev((10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)).astype(np.float32))
    back = [None, None]

    def step():
        ctx.paged_rope_kv_store(c.kv, c.pages, b, q, k, v, nh, hd, inv, True, q_out=qr)
        ctx.paged_attention(c.kv, c.pages, b, qr, nh, out=o)
        back[:] = ctx.paged_kv_read(c.kv, c.pages, b)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ctx.set_stream(torch.cuda.current_stream())
            step()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    held = list(back)
    for i, (ln, rows) in enumerate((([700, 300, 900], [1, 129, 0]), ([700, 1, 33], [70, 1, 33]), ([0, 5, 0], [0, 5, 0]),
                                    ([650, 290, 880], [30, 50, 50]))):
        lens.copy_(_dev(ln, np.int32))
        rs.copy_(_dev(np.concatenate([[0], np.cumsum(rows)]), np.int32))
        n = sum(rows)
        for x in (q, k, v):
            x.normal_(generator=g)
        o.fill_(5.0)
        qr.fill_(6.0)
        keep = c.pages.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (o, qr, c.pages, held[0][:n], held[1][:n])]
        assert (o[n:] == 5.0).all() and (qr[n:] == 6.0).all()
        o.fill_(5.0)
        qr.fill_(6.0)
        c.pages.copy_(keep)
        step()
        torch.cuda.synchronize()
        for x, y in zip(got, (o, qr, c.pages, back[0][:n], back[1][:n])):
            assert torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8)), i


def test_two_graphs_of_one_context_in_turn(ctx):  # noqa: F811
    """A decode step and a prompt chunk captured into two graphs, replayed in turn on one stream: they share the
    workspace that split rows are joined in."""
    import torch

    nh, nkv, hd = 8, 1, 128
    c = Cache(ctx, F16, nkv, hd, 256, [30000, 5000], 10)
    g = np.random.default_rng(10)
    calls = []
    for rows, lens in ((None, [30000, 5000]), ([200, 3], [29000, 4000])):
        q = _dev(g.standard_normal((2 if rows is None else 203, nh * hd)).astype(np.float32))
        b, o = c.batch(rows, lens=lens), torch.zeros_like(q)
        want = ctx.paged_attention(c.kv, c.pages, b, q, nh).clone()
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(graph):
                ctx.set_stream(torch.cuda.current_stream())
                ctx.paged_attention(c.kv, c.pages, b, q, nh, out=o)
        finally:
            ctx.set_stream(torch.cuda.current_stream())
        calls.append((graph, o, want, b, q))
    for _ in range(5):
        for graph, o, want, b, q in calls:
            o.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for graph, o, want, b, q in calls:
            assert torch.equal(o, want)
            assert torch.equal(ctx.paged_attention(c.kv, c.pages, b, q, nh), want)
