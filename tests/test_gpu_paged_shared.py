"""kmoe_paged_attention_shared against plain 64-bit attention of every sequence by
itself: groups of all kinds beside sequences of their own, single rows and chunks,
pages that are missing, values that are not finite, captured calls, refusals."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0, KmoeError, PagedGroups, PagedKV
from tests.test_gpu_paged import Cache, _close, _dev, _reference, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0]


def _shared(ctx, t, nkv, hd, page, lens, start, pages, seed, **kw):  # noqa: F811
    """A cache whose groups' members hold the leading pages of the longest of them (those of a shorter one would end
    before the shared positions do)."""
    c = Cache(ctx, t, nkv, hd, page, lens, seed, **kw)
    for i, p in enumerate(pages):
        members = range(start[i], start[i + 1])
        src = max(members, key=lambda b: lens[b], default=0)
        for b in members:
            n = min(p * page, lens[b])
            c.table[b, :p] = c.table[src, :p]
            for h in (c.hk, c.hv):
                h[b][:n] = h[src][:n]
    return c


def _attend(c, q, nh, start, pages, rows=None, out=None, batch=None, always=True):
    import torch

    g = c.ctx.paged_groups(_dev(start, np.int32), _dev(pages, np.int32), always=always)
    o = c.ctx.paged_attention_shared(c.kv, c.pages, batch or c.batch(rows), g, _dev(q.reshape(len(q), -1)), nh, out=out)
    torch.cuda.synchronize()
    return o.cpu().numpy()


def _check(c, nh, start, pages, rows=None, seed=0, **kw):
    S = len(c.lens) if rows is None else sum(rows)
    q = np.random.default_rng(seed).standard_normal((S, nh, c.kv.head_dim)).astype(np.float32)
    ref, tol, _ = _reference(c, q, rows, nh, **kw)
    # joining the two parts: a weight and its mean are rounded by three products, a sum and a quotient more
    _close(_attend(c, q, nh, start, pages, rows), ref, tol * (1 + 8 / 64))
    return q


# (lens, group starts, shared pages per group, at pages of 32 positions)
FORMS = [
    ([70, 80], [0, 2], [2]),                                              # the smallest group
    ([65] * 5, [0, 5], [2]),                                              # one position of their own
    ([40, 70, 99, 64, 33, 130, 97, 98, 1], [1, 3, 4, 8], [2, 7, 1]),      # groups, one of one, sequences before and behind
    ([200, 150, 96, 97, 300, 100], [0, 6], [3]),                          # the third one's row lies inside the shared pages
    ([50, 60, 70], [0, 3], [0]),                                          # nothing in common
    ([31, 32, 33], [0, 3], [1]),                                          # rows at the border
    ([10, 20, 30], [0, 0, 3, 3], [1, 1, 1]),                              # groups without sequences, pages past the lengths
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 64), (8, 2, 128), (16, 1, 64), (6, 3, 128)])
def test_single_rows(ctx, t, form, nh, nkv, hd):  # noqa: F811
    lens, start, pages = FORMS[form]
    c = _shared(ctx, t, nkv, hd, 32, lens, start, pages, form, extra_cols=form % 3)
    _check(c, nh, start, pages)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("page", [64, 256])
@pytest.mark.parametrize("rows", [[3, 3, 3, 3, 3, 3], [1, 40, 0, 7, 100, 2], [0, 0, 5, 0, 1, 0]])
def test_chunks(ctx, t, page, rows):  # noqa: F811
    """Several rows per sequence, none of some; the first group's second chunk reaches into the shared pages."""
    start, pages = [0, 3, 5], [2, 1]
    base = [2 * page + 50, 2 * page + 30, 2 * page + 60, page + 9, page + 120, 90]
    c = _shared(ctx, t, 2, 64, page, base, start, pages, page + sum(rows))
    _check(c, 6, start, pages, rows)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("members,shared,hd", [(64, 30, 128), (33, 90, 64), (3, 400, 128)])
def test_long_prefixes_split_among_the_work_groups(ctx, t, members, shared, hd):  # noqa: F811
    lens = [shared * 32 + 1 + 7 * i % 90 for i in range(members)]
    c = _shared(ctx, t, 2, hd, 32, lens, [0, members], [shared], members, spare=1)
    _check(c, 8, [0, members], [shared])


def test_many_groups(ctx):  # noqa: F811
    """More groups than a work-group has threads; sizes 1 .. 4."""
    rng = np.random.default_rng(5)
    start = np.concatenate([[3], 3 + np.cumsum(rng.integers(1, 5, 300))]).tolist()
    pages = rng.integers(0, 4, 300).tolist()
    lens = (32 * 3 + rng.integers(1, 60, start[-1] + 2)).tolist()
    c = _shared(ctx, F16, 1, 64, 32, lens, start, pages, 6)
    _check(c, 2, start, pages)


@pytest.mark.parametrize("start,pages", [([-7, 2, 99], [2, 10 ** 9]), ([0, 4], [-3]), ([4, 4], [1]), ([-9, -2], [1]), ([7, 12], [2]),
                                         ([2 ** 31 - 1, 2 ** 31 - 1], [2 ** 31 - 1]), ([-2 ** 31, 2], [2])])
def test_entries_past_the_batch_or_the_table_are_cut_off(ctx, start, pages):  # noqa: F811
    lens = [70, 80, 90, 100]
    c = _shared(ctx, F16, 2, 64, 32, lens, [0, 2, 4], [2, 0], 7)
    _check(c, 4, start, pages)


@pytest.mark.parametrize("start,pages", [([0, 3, -2 ** 31], [2, 1]), ([3, -2 ** 31], [2]), ([2 ** 31 - 1, -2 ** 31], [1]), ([3, 1], [2])])
def test_a_group_that_ends_before_it_begins_is_none(ctx, start, pages):  # noqa: F811
    c = _shared(ctx, F16, 2, 64, 32, [70, 80, 90, 100], [0, 3], [2], 7)
    _check(c, 4, start, pages)


@pytest.mark.parametrize("nh,nkv,hd,most", [(4, 2, 64, 1), (4, 2, 128, 1), (16, 1, 64, 3), (16, 1, 128, 3)])
def test_as_many_sequences_as_a_call_takes(ctx, nh, nkv, hd, most):  # noqa: F811
    """4096 sequences, in groups of every size up to 60 with one or two pages of 32 in common."""
    rng = np.random.default_rng(hd + most)
    lens = rng.integers(most, 110, 4096).tolist()
    rows = None if most == 1 else rng.integers(1, most + 1, 4096).tolist()
    if rows:
        lens = [max(n, r) for n, r in zip(lens, rows)]
    start = np.unique(np.concatenate([[0, 4096], np.cumsum(rng.integers(1, 61, 200))]).clip(0, 4096)).tolist()
    pages = rng.integers(0, 3, len(start) - 1).tolist()
    c = _shared(ctx, F16, nkv, hd, 32, lens, start, pages, 14)
    S = 4096 if rows is None else sum(rows)
    q = rng.standard_normal((S, nh, hd)).astype(np.float32)
    got = _attend(c, q, nh, start, pages, rows).reshape(S, nh, hd)
    assert np.isfinite(got).all()
    pick = [0, 1, 255, 256, 257, 2048, 4094, 4095] + rng.integers(0, 4096, 60).tolist()
    rs = np.concatenate([[0], np.cumsum([1] * 4096 if rows is None else rows)])
    at = np.concatenate([np.arange(rs[b], rs[b + 1]) for b in pick])
    sub = SimpleNamespace(kv=c.kv, lens=[lens[b] for b in pick], hk=[c.hk[b] for b in pick], hv=[c.hv[b] for b in pick])
    ref, tol, _ = _reference(sub, q[at], None if rows is None else [rows[b] for b in pick], nh)
    _close(got[at], ref, tol * (1 + 8 / 64))


def test_as_many_groups_as_sequences(ctx):  # noqa: F811
    """4096 groups, two thousand of them of two sequences, the others empty."""
    lens, start = [40 + i % 50 for i in range(4096)], np.repeat(np.arange(0, 4097, 2), 2)[:4097].tolist()
    pages = [1] * 4096
    c = _shared(ctx, F16, 1, 64, 32, lens, start, pages, 15)
    q = np.random.default_rng(5).standard_normal((4096, 2, 64)).astype(np.float32)
    got = _attend(c, q, 2, start, pages).reshape(4096, 2, 64)
    pick = list(range(0, 4096, 73))
    sub = SimpleNamespace(kv=c.kv, lens=[lens[b] for b in pick], hk=[c.hk[b] for b in pick], hv=[c.hv[b] for b in pick])
    ref, tol, _ = _reference(sub, q[pick], None, 2)
    _close(got[pick], ref, tol * (1 + 8 / 64))


@pytest.mark.parametrize("t", TYPES)
def test_missing_pages(ctx, t):  # noqa: F811
    """Pages of the shared part, of a sequence's own, and all of both that name no page."""
    lens, start, pages = [130, 140, 150, 160], [0, 4], [3]
    c = _shared(ctx, t, 2, 64, 32, lens, start, pages, 8)
    hidden = [np.zeros(n, bool) for n in lens]
    c.table[:, 1] = -1
    for b in range(4):
        hidden[b][32:64] = True
    c.table[2, 3:] = 10 ** 6
    hidden[2][96:] = True
    _check(c, 4, start, pages, hidden=hidden)
    c.table[:, :3] = -1
    for h in hidden:
        h[:96] = True
    _check(c, 4, start, pages, hidden=hidden)  # (the third one's row sees nothing: zeros)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("what", ["v_nan", "v_inf", "k_nan", "k_-inf", "k_all_-inf", "own_-inf", "everything_-inf"])
def test_not_finite(ctx, t, what):  # noqa: F811
    """What kmoe_paged_attention gives, element by element: NaN and infinities where it has them."""
    import torch

    page, lens, start, pages, nh, nkv, hd = 32, [75, 80, 90, 70], [0, 3], [2], 4, 2, 64
    c = _shared(ctx, F16, nkv, hd, page, lens, start, pages, 9)  # (f16 pages hold infinities as they are)
    if t == Q8_0:
        c = _shared(ctx, Q8_0, nkv, hd, page, lens, start, pages, 9)
    k = [x.copy() for x in c.k]
    v = [x.copy() for x in c.v]
    for x in (k, v):
        for b in (1, 2):
            x[b][:64] = x[0][:64]
    at = {"own_-inf": slice(64, None), "everything_-inf": slice(0, None), "k_all_-inf": slice(0, 64)}.get(what, slice(40, 41))
    val = np.nan if "nan" in what else np.inf if what == "v_inf" else -np.inf
    for b in range(3):
        if what[0] == "v":
            v[b][at, 1, 5] = val
        else:
            k[b][at, 1] = 0
            k[b][at, 1, 0] = val
    # the store writes shared pages several times, the same values each time
    for b in range(4):
        bt = ctx.paged_batch(_dev(c.table[b:b + 1]), _dev(lens[b:b + 1], np.int32), _dev([0, lens[b]], np.int32), lens[b])
        ctx.paged_kv_store(c.kv, c.pages, bt, _dev(k[b].reshape(lens[b], -1)), _dev(v[b].reshape(lens[b], -1)))
    q = np.random.default_rng(1).standard_normal((4, nh, hd)).astype(np.float32)
    q[:, :, 0] = np.abs(q[:, :, 0]) + 0.1
    want = ctx.paged_attention(c.kv, c.pages, c.batch(), _dev(q.reshape(4, -1)), nh)
    torch.cuda.synchronize()
    want, got = want.cpu().numpy(), _attend(c, q, nh, start, pages)
    assert np.array_equal(np.isnan(want), np.isnan(got)) and np.array_equal(np.isinf(want), np.isinf(got))
    f = np.isfinite(want)
    assert np.abs(want[f] - got[f]).max(initial=0) <= 2e-6 and np.isfinite(got[3]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,shared", [(128, 48), (64, 96)])
def test_groups_are_read_once_where_that_saves_enough(ctx, t, hd, shared):  # noqa: F811
    """Besides groups that are not worth it, and batches of them alone; without `always`."""
    lens = [shared * 32 + 1 + i % 40 for i in range(48)] + [40, 50, 60, 1500]
    for start, pages in (([0, 48, 51], [shared, 1]), ([48, 51], [1]), ([0, 2, 51], [1, 1]), ([0, 0, 48], [shared, shared])):
        c = _shared(ctx, t, 8, hd, 32, lens, start, pages, 16)
        q = np.random.default_rng(6).standard_normal((len(lens), 16, hd)).astype(np.float32)
        g = _attend(c, q, 16, start, pages, always=False)
        pick = [0, 1, 30, 47, 48, 50, 51]
        sub = SimpleNamespace(kv=c.kv, lens=[lens[b] for b in pick], hk=[c.hk[b] for b in pick], hv=[c.hv[b] for b in pick])
        ref, tol, _ = _reference(sub, q[pick], None, 16)
        _close(g.reshape(q.shape)[pick], ref, tol * (1 + 8 / 64))
        whole = ctx.paged_attention(c.kv, c.pages, c.batch(), _dev(q.reshape(len(q), -1)), 16).cpu().numpy()
        g = g.reshape(whole.shape)
        # 47 rows of 8 kv heads save 16000 (heads of 64: 32000) tiles' work, the others next to nothing
        assert np.array_equal(g, whole) == (pages[0] != shared and pages[-1] != shared)


def test_rows_behind_the_last_sequence_and_given_outputs(ctx):  # noqa: F811
    import torch

    lens, start, pages, rows = [70, 80, 66], [0, 3], [2], [2, 1, 2]
    c = _shared(ctx, F16, 2, 64, 32, lens, start, pages, 10)
    q = np.random.default_rng(2).standard_normal((9, 4, 64)).astype(np.float32)
    out = torch.full((9, 256), 7.0, device="cuda")
    got = _attend(c, q, 4, start, pages, out=out, batch=c.batch(rows, s_rows=9))
    assert (got[5:] == 7).all() and (got[:5] != 7).all()
    assert ctx.paged_attention_shared(c.kv, c.pages, c.batch([0, 0, 0]), ctx.paged_groups(_dev(start, np.int32), _dev(pages, np.int32)),
                                      torch.empty((0, 256), device="cuda"), 4).shape == (0, 256)


def test_captured_calls_follow_the_arrays(ctx):  # noqa: F811
    """Replayed with other lengths, tables and groups, on a stream of the capture's, with eager calls between."""
    import torch

    forms = [([300, 280, 310, 270], [0, 2, 4], [8, 5]), ([300, 257, 310, 259], [0, 4, 4], [8, 3]), ([20, 280, 310, 270], [1, 1, 3], [1, 6])]
    cs = [_shared(ctx, F16, 2, 128, 32, *f, 11 + i) for i, f in enumerate(forms)]
    q = np.random.default_rng(3).standard_normal((4, 8, 128)).astype(np.float32)
    cols = max(c.cols for c in cs)
    pages = torch.empty((max(c.pages.shape[0] for c in cs), cs[0].kv.page_bytes), dtype=torch.uint8, device="cuda")
    table, lens = torch.full((4, cols), -1, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    start, shared = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    dq, out = _dev(q.reshape(4, -1)), torch.empty((4, 1024), device="cuda")
    batch, groups = ctx.paged_batch(table, lens), ctx.paged_groups(start, shared, always=True)
    ctx.paged_attention_shared(cs[0].kv, pages, batch, groups, dq, 8, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.paged_attention_shared(cs[0].kv, pages, batch, groups, dq, 8, out=out)
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in (0, 1, 2, 1, 0):
        c, (ln, st, pg) = cs[i], forms[i]
        pages[:c.pages.shape[0]] = c.pages
        table.fill_(-1)
        table[:, :c.cols] = _dev(c.table)
        for d, x in ((lens, ln), (start, st), (shared, pg)):
            d.copy_(_dev(x, np.int32))
        graph.replay()
        torch.cuda.synchronize()
        ref, tol, _ = _reference(c, q, None, 8)
        _close(out.cpu().numpy(), ref, tol * (1 + 8 / 64))
        assert torch.equal(out, ctx.paged_attention_shared(cs[0].kv, pages, batch, groups, dq, 8))


def test_streams_take_turns(ctx):  # noqa: F811
    """Calls on two streams of one context share its workspaces."""
    import torch

    lens, start, pages = [2000 + i for i in range(8)], [0, 8], [60]
    c = _shared(ctx, F16, 2, 128, 32, lens, start, pages, 12)
    g, q = ctx.paged_groups(_dev(start, np.int32), _dev(pages, np.int32), always=True), _dev(np.random.default_rng(4).standard_normal((2, 8, 1024)))
    qs, b = [x.float().contiguous() for x in q], c.batch()
    want = [ctx.paged_attention_shared(c.kv, c.pages, b, g, x, 8).clone() for x in qs]
    torch.cuda.synchronize()
    ss, outs = [torch.cuda.Stream() for _ in range(2)], []
    try:
        for i in range(20):
            ctx.set_stream(ss[i % 2])
            outs.append((ctx.paged_attention_shared(c.kv, c.pages, b, g, qs[i % 2], 8, out=torch.empty_like(want[0])), want[i % 2]))
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(torch.cuda.current_stream())
    assert all(torch.equal(x, y) for x, y in outs)


def test_refusals(ctx):  # noqa: F811
    import torch

    lens, start, pages = [70, 80], [0, 2], [2]
    c = _shared(ctx, F16, 2, 64, 32, lens, start, pages, 13)
    g, q = ctx.paged_groups(_dev(start, np.int32), _dev(pages, np.int32)), torch.zeros((2, 256), device="cuda")
    call = lambda **k: ctx.paged_attention_shared(**{**dict(kv=c.kv, pages=c.pages, batch=c.batch(), groups=g, q=q, n_head=4), **k})  # noqa: E731
    for bad in (dict(q=q.half()), dict(q=q[:1]), dict(q=q.t()), dict(out=q[:1]), dict(q=q.cpu()), dict(pages=c.pages.cpu())):
        with pytest.raises(ValueError):
            call(**bad)
    for st, pg in ((_dev([0, 2]), _dev([2], np.int32)), (_dev([0, 2], np.int32), _dev([2, 1], np.int32)),
                   (_dev([0, 2], np.int32).cpu(), _dev([2], np.int32))):
        with pytest.raises(ValueError):
            ctx.paged_groups(st, pg)
    for bad in (dict(out=q), dict(n_head=3, q=torch.zeros((2, 192), device="cuda")), dict(groups=PagedGroups(4097, g.start, g.pages)),
                dict(groups=PagedGroups(-1, g.start, g.pages)), dict(groups=PagedGroups(1, None, g.pages)), dict(groups=PagedGroups(1, g.start, None))):
        with pytest.raises(KmoeError) as e:
            call(**bad)
        assert e.value.status == -1
    with pytest.raises(KmoeError) as e:
        call(n_head=34, q=torch.zeros((2, 34 * 64), device="cuda"))
    assert e.value.status == -2
    assert ctx.lib.kmoe_paged_attention_shared(ctx.h, C.byref(c.kv.desc(c.pages)), c.pages.data_ptr(), C.byref(c.batch()), None,
                                               q.data_ptr(), 4, q.data_ptr() + 4096) == -1
    # 2^21 rows by heads are the most: 131072 rows of 16 heads go, one more does not
    kv = PagedKV(F16, 1, 64, 32)
    n = (1 << 21) // 16 + 1
    b = ctx.paged_batch(_dev([[0]], np.int32), _dev([1], np.int32), _dev([0, 1], np.int32), n)
    big = torch.zeros((n, 16 * 64), device="cuda")
    p = torch.zeros((1, kv.page_bytes), dtype=torch.uint8, device="cuda")
    with pytest.raises(KmoeError) as e:
        ctx.paged_attention_shared(kv, p, b, ctx.paged_groups(_dev([0, 1], np.int32), _dev([1], np.int32)), big, 16)
    assert e.value.status == -2
    # no groups at all: kmoe_paged_attention
    assert torch.equal(call(groups=ctx.paged_groups(_dev([0], np.int32), _dev([], np.int32)), q=q + 1),
                       ctx.paged_attention(c.kv, c.pages, c.batch(), q + 1, 4))
    torch.cuda.synchronize()
