"""Bounds of pages and attention over the pages that they select (kmoe_paged_select.hip)
against plain 64-bit forms: single rows and chunks, contexts that several work-groups
score, equal scores, missing pages, values that are not finite, captured calls, refusals."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0, KmoeError, PagedKV
from tests.test_gpu_paged import Cache, _close, _dev, _reference, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0]


def _bounds_of(c, lens=None):
    """[n_pages, nkv, 2, hd] f16 of the sequences' pages; NaN elsewhere."""
    kv = c.kv
    out = np.full((c.pages.shape[0], kv.n_kv, 2, kv.head_dim), np.nan, np.float16)
    for b, n in enumerate(c.lens if lens is None else lens):
        for j in range(-(-n // kv.page)):
            k = c.hk[b][j * kv.page:min(n, (j + 1) * kv.page)]
            if 0 <= c.table[b, j] < len(out):
                with np.errstate(invalid="ignore"):
                    out[c.table[b, j], :, 0] = np.fmin.reduce(k, axis=0)
                    out[c.table[b, j], :, 1] = np.fmax.reduce(k, axis=0)
    return out


def _fresh(c):
    import torch

    return torch.full((c.pages.shape[0], c.kv.n_kv, 2, c.kv.head_dim), float("nan"), dtype=torch.float16, device="cuda")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nkv,hd,page,lens", [(1, 64, 32, [1]), (4, 128, 64, [37, 64, 65, 1, 200]), (3, 64, 256, [255, 256, 257, 16]),
                                              (2, 128, 128, [300, 5, 129]), (8, 64, 32, [31, 32, 33, 1000])])
def test_bounds_of_whole_sequences(ctx, t, nkv, hd, page, lens):  # noqa: F811
    """All rows at once; positions past a length hold NaN and must not be read."""
    c = Cache(ctx, t, nkv, hd, page, lens, 1, extra_cols=1, scale=3.0)
    got = ctx.paged_bounds(c.kv, c.pages, c.batch(lens), _fresh(c)).cpu().numpy()
    assert np.array_equal(got, _bounds_of(c), equal_nan=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [None, [1, 1, 1, 1], [0, 70, 1, 3], [5, 0, 0, 64], [33, 65, 1, 2]])
def test_bounds_of_new_rows(ctx, t, rows):  # noqa: F811
    """Only the pages that the batch's rows lie on are written, each over all of its positions."""
    lens, page = [70, 130, 64, 33], 32
    c = Cache(ctx, t, 2, 64, page, lens, 2)
    got = ctx.paged_bounds(c.kv, c.pages, c.batch(rows), _fresh(c)).cpu().numpy()
    want = _bounds_of(c)
    for b, n in enumerate(lens):
        r = 1 if rows is None else rows[b]
        for j in range(-(-n // page)):
            if r == 0 or j < (n - r) // page:
                want[c.table[b, j]] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


def test_bounds_edges(ctx):  # noqa: F811
    """Lengths of zero and below the rows, past the table, missing pages, NaN and infinite keys, Q8_0 past f16's range."""
    import torch

    c = Cache(ctx, F16, 1, 64, 32, [40, 50, 60], 3, extra_cols=0)
    want = _bounds_of(c)
    b = ctx.paged_batch(_dev(c.table), _dev([0, -5, 10 ** 9], np.int32))
    assert torch.isnan(ctx.paged_bounds(c.kv, c.pages, b, _fresh(c))).all()
    b = ctx.paged_batch(_dev(c.table), _dev([40, 50, 60], np.int32), _dev([0, 100, 100, 230], np.int32), 230)  # more rows than positions
    got = ctx.paged_bounds(c.kv, c.pages, b, _fresh(c)).cpu().numpy()
    want[c.table[1]] = np.nan
    assert np.array_equal(got, want, equal_nan=True)
    t = c.table.copy()
    t[0, 1], t[2, 0] = -1, 10 ** 6
    got = ctx.paged_bounds(c.kv, c.pages, c.batch([40, 0, 60], table=t), _fresh(c)).cpu().numpy()
    want[[c.table[0, 1], c.table[2, 0]]] = np.nan
    assert np.array_equal(got, want, equal_nan=True)
    k = np.zeros((3, 64), np.float32)
    k[0, :3], k[1, :3], k[2, :3] = [np.nan, np.inf, 1], [2, 0, -np.inf], [-1, 5, 0]
    for ty, z in ((F16, 1.0), (Q8_0, 1.0e7)):
        kv = PagedKV(ty, 1, 64, 32)
        pages = torch.zeros((1, kv.page_bytes), dtype=torch.uint8, device="cuda")
        b = ctx.paged_batch(_dev([[0]], np.int32), _dev([3], np.int32), _dev([0, 3], np.int32), 3)
        x = k if ty == F16 else np.where(np.isfinite(k), k, 0).astype(np.float32) * np.float32(z)
        ctx.paged_kv_store(kv, pages, b, _dev(x), _dev(x))
        got = ctx.paged_bounds(kv, pages, b, torch.empty((1, 1, 2, 64), dtype=torch.float16, device="cuda")).cpu().numpy()[0, 0, :, :3]
        if ty == F16:
            assert np.array_equal(got, np.array([[-1, 0, -np.inf], [2, np.inf, 1]], np.float16))
        else:
            assert np.isfinite(got).all() and np.abs(got).max() == 65504


# ------------------------------------------------------------------ attention

def _select(c, q, rows, nh, n_select, n_first, bounds):
    """Per sequence the positions [rows, nkv, n] that are hidden because their pages are not chosen, by the definition."""
    kv, hidden, at = c.kv, [], 0
    G = nh // kv.n_kv
    for b, n in enumerate(c.lens):
        r = 1 if rows is None else rows[b]
        h = np.ones((r, kv.n_kv, n), bool)
        for i in range(r):
            pos = n - r + i
            if pos < 0:
                continue
            own, seen = pos // kv.page, []
            ids = [c.table[b, j] if j < c.cols and 0 <= c.table[b, j] < len(bounds) else -1 for j in range(own + 1)]
            for g in range(kv.n_kv):
                seen = [own] if ids[own] >= 0 else []
                seen += [j for j in range(min(n_first, own)) if ids[j] >= 0]
                rest = [j for j in range(n_first, own) if ids[j] >= 0]
                x = q[at + i, g * G:(g + 1) * G].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = [np.maximum(x * bounds[ids[j], g, 0].astype(np.float64), x * bounds[ids[j], g, 1].astype(np.float64)).sum() for j in rest]
                s = np.where(np.isnan(s), np.inf, s) if len(s) else np.zeros(0)
                best = np.argsort(-s, kind="stable")[:max(0, n_select - len(seen))]
                for j in seen + [rest[x] for x in best]:
                    h[i, g, j * kv.page:(j + 1) * kv.page] = False
        hidden.append(h)
        at += r
    return hidden


def _reference_selected(c, q, rows, nh, hidden):
    """_reference of test_gpu_paged per row and kv head, each over what it sees."""
    nkv, hd, at = c.kv.n_kv, c.kv.head_dim, 0
    S, G = len(q), nh // nkv
    out, tol = np.zeros((S, nh, hd)), np.zeros((S, nh, hd))

    class One:
        pass

    for b, n in enumerate(c.lens):
        r = 1 if rows is None else rows[b]
        for i in range(r):
            for g in range(nkv):
                o = One()
                o.kv, end = PagedKV(c.kv.type, 1, hd, c.kv.page), max(0, n - r + i + 1)
                o.lens, o.hk, o.hv = [end], [c.hk[b][:end, g:g + 1]], [c.hv[b][:end, g:g + 1]]
                y, e, _ = _reference(o, q[at:at + 1, g * G:(g + 1) * G], None, G, hidden=[hidden[b][i, g, :end]])
                out[at, g * G:(g + 1) * G], tol[at, g * G:(g + 1) * G] = y[0], e[0]
            at += 1
    return out, tol


def _attend(c, q, nh, n_select, n_first=0, rows=None, bounds=None, batch=None, out=None):
    import torch

    bounds = _dev(np.nan_to_num(_bounds_of(c), nan=0.0), np.float16) if bounds is None else bounds
    o = c.ctx.paged_attention_selected(c.kv, c.pages, bounds, batch or c.batch(rows), _dev(q.reshape(len(q), -1)), nh, n_select,
                                       n_first, out=out)
    torch.cuda.synchronize()
    return o.cpu().numpy()


def _check(c, nh, n_select, n_first=0, rows=None, seed=0):
    S = len(c.lens) if rows is None else sum(rows)
    q = np.random.default_rng(seed).standard_normal((S, nh, c.kv.head_dim)).astype(np.float32)
    hidden = _select(c, q, rows, nh, n_select, n_first, _bounds_of(c))
    ref, tol = _reference_selected(c, q, rows, nh, hidden)
    _close(_attend(c, q, nh, n_select, n_first, rows), ref, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n_select,n_first", [(1, 0), (2, 0), (2, 1), (3, 1), (5, 2), (7, 6)])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 64), (8, 2, 128), (16, 1, 64), (6, 3, 128)])
def test_single_rows(ctx, t, n_select, n_first, nh, nkv, hd):  # noqa: F811
    c = Cache(ctx, t, nkv, hd, 32, [1, 32, 33, 64, 290, 257, 100, 500], n_select, extra_cols=n_first)
    _check(c, nh, n_select, n_first)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("page", [64, 128, 256])
def test_chunks(ctx, t, page):  # noqa: F811
    """Every row of a chunk has pages of its own; sequences without rows; over a thousand rows by kv heads."""
    lens, rows = [7 * page + 3, 5 * page, 90, 3 * page + 1], [40, 0, 90, 3]
    c = Cache(ctx, t, 2, 64, page, lens, page)
    _check(c, 4, 3, 1, rows)


def test_more_rows_than_a_launch_takes(ctx):  # noqa: F811
    c = Cache(ctx, F16, 4, 64, 32, [400, 60, 350], 5)
    _check(c, 4, 4, 1, [330, 0, 170])


@pytest.mark.parametrize("lens,rows,extra", [([900, 60, 500], [800, 0, 300], 0), ([600, 40], [170, 1], 1 << 14), ([40 + i % 60 for i in range(1100)], None, 0)])
def test_more_rows_than_a_choice_takes(ctx, lens, rows, extra):  # noqa: F811
    """Over 4096 rows by kv heads, or 2^22 by the table's columns: several launches of the choice, too."""
    c = Cache(ctx, F16, 4, 64, 32, lens, 8, extra_cols=extra)
    _check(c, 4, 3, 1, rows)


def test_more_kv_heads_than_rows_of_a_launch(ctx):  # noqa: F811
    """One row, and one chunk, of 1500 kv heads; contexts that two work-groups score."""
    c = Cache(ctx, F16, 1500, 64, 32, [32 * 4 + 3, 32 * 5], 6)
    _check(c, 1500, 2, 0)
    _check(c, 1500, 3, 1, [2, 1])
    c = Cache(ctx, F16, 300, 64, 32, [32 * 130 + 3], 7)
    _check(c, 300, 4, 1)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n_select", [2, 40, 700])
def test_contexts_that_several_work_groups_score(ctx, t, n_select):  # noqa: F811
    """511, 512, 513 and more columns before a row's own."""
    lens = [32 * m + x for m, x in ((511, 32), (512, 1), (512, 32), (513, 5), (1030, 7), (3, 1))]
    c = Cache(ctx, t, 1, 64, 32, lens, n_select)
    for i in range(3):  # the counters are zero again after every call
        _check(c, 2, n_select, 1, seed=i)


def test_equal_scores_go_to_the_lower_position(ctx):  # noqa: F811
    """Pages of four contents only, their values apart: which of the equal ones is read shows."""
    import torch

    c = Cache(ctx, F16, 2, 64, 32, [32 * 600 + 10], 6)
    kinds = np.random.default_rng(7).integers(0, 4, 601)
    content = np.random.default_rng(8).standard_normal((4, 32, 2, 64)).astype(np.float32)
    c.k[0] = np.concatenate([content[x] for x in kinds])[:c.lens[0]]
    c.hk[0] = c.k[0].astype(np.float16).astype(np.float64)
    ctx.paged_kv_store(c.kv, c.pages, c.batch(c.lens), _dev(c.k[0].reshape(c.lens[0], -1)), _dev(c.v[0].reshape(c.lens[0], -1)))
    torch.cuda.synchronize()
    for n_select in (2, 30, 200, 470, 600):
        _check(c, 4, n_select, 0, seed=n_select)
    q = np.zeros((1, 4, 64), np.float32)  # all scores are 0
    for n_select in (3, 300):
        hidden = _select(c, q, None, 4, n_select, 0, _bounds_of(c))
        assert not hidden[0][0, 0, :32 * (n_select - 1)].any()
        ref, tol = _reference_selected(c, q, None, 4, hidden)
        _close(_attend(c, q, 4, n_select), ref, tol)


@pytest.mark.parametrize("t", TYPES)
def test_missing_pages(ctx, t):  # noqa: F811
    """Of the first ones, the middle, a row's own, and all."""
    c = Cache(ctx, t, 2, 64, 32, [300, 310, 320, 290, 30], 9)
    full = c.table.copy()
    for cols in ([0], [4], [9], [0, 1, 2, 5, 9], list(range(9)), list(range(10))):
        c.table = full.copy()
        c.table[:4, cols] = -1
        c.table[1, cols] = 10 ** 6
        for n_select, n_first in ((3, 1), (2, 0), (6, 3)):
            _check_missing(c, n_select, n_first)


def _check_missing(c, n_select, n_first):
    q = np.random.default_rng(n_select).standard_normal((5, 4, 64)).astype(np.float32)
    want = _bounds_of(c)
    hidden = _select(c, q, None, 4, n_select, n_first, want)
    ref, tol = _reference_selected(c, q, None, 4, hidden)
    _close(_attend(c, q, 4, n_select, n_first), ref, tol)


def test_lengths_past_the_table_and_below_the_rows(ctx):  # noqa: F811
    """A row past the table sees whole pages only; one without a position sees nothing."""
    c = Cache(ctx, F16, 1, 64, 32, [128, 128, 100, 90], 10)
    q = np.random.default_rng(1).standard_normal((6, 2, 64)).astype(np.float32)
    b = ctx.paged_batch(_dev(c.table), _dev([10 ** 6, 2 ** 31 - 1, 1, 0], np.int32), _dev([0, 1, 2, 5, 6], np.int32), 6)
    got = _attend(c, q, 2, 2, 1, batch=b).reshape(6, 2, 64)
    c.lens, rows = [128, 128], None
    hidden = _select(c, q[:2], rows, 2, 2, 1, _bounds_of(c))
    ref, tol = _reference_selected(c, q[:2], rows, 2, hidden)
    _close(got[:2], ref, tol)
    assert (got[[2, 3, 5]] == 0).all()
    _close(got[4:5], np.broadcast_to(c.hv[2][:1, 0], (1, 2, 64)), np.full((1, 2, 64), 1e-6))


def test_as_many_pages_as_there_are(ctx):  # noqa: F811
    """Fewer pages than n_select: all of them; n_select of the table's width: kmoe_paged_attention's bits."""
    import torch

    c = Cache(ctx, Q8_0, 2, 128, 64, [300, 500, 64], 11)
    _check(c, 8, c.cols - 1, 1)
    q = np.random.default_rng(2).standard_normal((3, 8, 128)).astype(np.float32)
    for n in (c.cols, 10 ** 6, 2 ** 31 - 1):
        got = _attend(c, q, 8, n, 3)
        assert np.array_equal(got, ctx.paged_attention(c.kv, c.pages, c.batch(), _dev(q.reshape(3, -1)), 8).cpu().numpy())
    torch.cuda.synchronize()


def test_not_finite(ctx):  # noqa: F811
    """A page with an infinite key scores best where q reaches for it; NaN in q or a score; NaN keys on pages that are
    not chosen reach nothing."""
    c = Cache(ctx, F16, 1, 64, 32, [330], 12)
    q = np.abs(np.random.default_rng(3).standard_normal((1, 1, 64))).astype(np.float32)
    k = c.k[0].copy()
    k[2 * 32 + 5, 0, 7] = np.inf
    ctx.paged_kv_store(c.kv, c.pages, c.batch([330]), _dev(k.reshape(330, -1)), _dev(c.v[0].reshape(330, -1)))
    c.hk[0] = k.astype(np.float16).astype(np.float64)
    b = _bounds_of(c)
    assert np.isinf(b).sum() == 1
    dense = ctx.paged_attention(c.kv, c.pages, c.batch(), _dev(q.reshape(1, -1)), 1).cpu().numpy()
    got = _attend(c, q, 1, 2)
    assert np.isnan(dense).any() == np.isnan(got).any()  # the infinite score's page is among the two
    nq = q.copy()
    nq[0, 0, 3] = np.nan
    assert np.isnan(_attend(c, nq, 1, 2)).all()
    zq = -q  # reaches for no large key: the page's lo bounds decide, and the infinity (a score of -inf) is not chosen first
    k[5 * 32 + 1] = np.nan
    ctx.paged_kv_store(c.kv, c.pages, c.batch([330]), _dev(k.reshape(330, -1)), _dev(c.v[0].reshape(330, -1)))
    c.hk[0] = k.astype(np.float16).astype(np.float64)
    hidden = _select(c, zq, None, 1, 2, 0, _bounds_of(c))
    if hidden[0][0, 0, 5 * 32 + 1] and hidden[0][0, 0, 2 * 32 + 5]:
        ref, tol = _reference_selected(c, zq, None, 1, hidden)
        _close(_attend(c, zq, 1, 2), ref, tol)


def test_scores_past_the_doubles_middle(ctx):  # noqa: F811
    """Scores of both signs over sixty powers of two and more: the ranges of the choice narrow from 64 bits to one."""
    import torch

    rng = np.random.default_rng(13)
    n_pages, kv = 700, PagedKV(F16, 1, 64, 32)
    c = Cache(ctx, F16, 1, 64, 32, [32 * n_pages], 13)
    bounds = np.zeros((c.pages.shape[0], 1, 2, 64), np.float16)
    e = rng.choice(np.concatenate([2.0 ** np.arange(-24, 15), -2.0 ** np.arange(-24, 15), [0.0]]), n_pages)
    bounds[c.table[0], 0, :, 0] = e[:, None]
    for scale in (1.0, 1.0e-30, 1.0e30):
        q = np.zeros((1, 1, 64), np.float32)
        q[0, 0, 0] = scale
        for n_select in (2, 100, 350, 600, 699):
            hidden = _select(c, q, None, 1, n_select, 0, bounds)
            q2 = q.copy()
            ref, tol = _reference_selected(c, q2, None, 1, hidden)
            got = _attend(c, q2, 1, n_select, bounds=_dev(bounds, np.float16))
            if scale < 1.0e20:
                _close(got, ref, tol)
    assert kv.page == c.kv.page
    torch.cuda.synchronize()


def test_rows_outside_the_sequences_are_left(ctx):  # noqa: F811
    import torch

    c = Cache(ctx, F16, 2, 64, 32, [200, 150, 180], 14)
    q = np.random.default_rng(4).standard_normal((12, 4, 64)).astype(np.float32)
    out = torch.full((12, 256), 7.0, device="cuda")
    b = ctx.paged_batch(_dev(c.table), _dev(c.lens, np.int32), _dev([3, 5, 5, 9], np.int32), 12)
    got = _attend(c, q, 4, 3, batch=b, out=out)
    assert (got[:3] == 7).all() and (got[9:] == 7).all() and (got[3:9] != 7).all()
    want = _attend(c, q[3:9], 4, 3, rows=[2, 0, 4])
    assert np.abs(got[3:9] - want).max() <= 1e-6
    b = ctx.paged_batch(_dev(c.table), _dev(c.lens, np.int32), _dev([12, 12, 12, 12], np.int32), 12)
    assert (_attend(c, q, 4, 3, batch=b, out=torch.full((12, 256), 7.0, device="cuda")) == 7).all()


def test_captured_calls_follow_the_lengths(ctx):  # noqa: F811
    """Bounds and attention captured together, replayed at other lengths with other queries."""
    import torch

    lens = [32 * 520 + 7, 700, 90]
    c = Cache(ctx, F16, 2, 64, 32, lens, 15)
    full_k, full_v = c.hk, c.hv
    bounds = _dev(np.nan_to_num(_bounds_of(c), nan=0.0), np.float16)
    ln, q, out = _dev(lens, np.int32), torch.zeros((3, 256), device="cuda"), torch.empty((3, 256), device="cuda")
    batch = ctx.paged_batch(_dev(c.table), ln)

    def step():
        ctx.paged_bounds(c.kv, c.pages, batch, bounds)
        ctx.paged_attention_selected(c.kv, c.pages, bounds, batch, q, 4, 6, 1, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ctx.set_stream(torch.cuda.current_stream())
            step()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i, ls in enumerate(([16647, 700, 90], [16385, 33, 90], [16000, 640, 1], [16640, 700, 64])):
        hq = np.random.default_rng(i).standard_normal((3, 4, 64)).astype(np.float32)
        ln.copy_(_dev(ls, np.int32))
        q.copy_(_dev(hq.reshape(3, -1)))
        graph.replay()
        torch.cuda.synchronize()
        c.lens, c.hk, c.hv = ls, [k[:n] for k, n in zip(full_k, ls)], [v[:n] for v, n in zip(full_v, ls)]
        hb = bounds.cpu().numpy()
        ref, tol = _reference_selected(c, hq, None, 4, _select(c, hq, None, 4, 6, 1, hb))
        _close(out.cpu().numpy(), ref, tol)
        assert torch.equal(out, ctx.paged_attention_selected(c.kv, c.pages, bounds, batch, q, 4, 6, 1))


def test_streams_take_turns(ctx):  # noqa: F811
    import torch

    c = Cache(ctx, F16, 2, 64, 32, [32 * 1100, 5000], 16)
    bounds, b = _dev(np.nan_to_num(_bounds_of(c), nan=0.0), np.float16), c.batch()
    qs = [_dev(np.random.default_rng(i).standard_normal((2, 256)).astype(np.float32)) for i in range(2)]
    want = [ctx.paged_attention_selected(c.kv, c.pages, bounds, b, q, 4, 20).clone() for q in qs]
    torch.cuda.synchronize()
    ss, outs = [torch.cuda.Stream() for _ in range(2)], []
    try:
        for i in range(20):
            ctx.set_stream(ss[i % 2])
            outs.append((ctx.paged_attention_selected(c.kv, c.pages, bounds, b, qs[i % 2], 4, 20, out=torch.empty_like(want[0])), want[i % 2]))
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(torch.cuda.current_stream())
    assert all(torch.equal(x, y) for x, y in outs)


def test_refusals(ctx):  # noqa: F811
    import torch

    c = Cache(ctx, F16, 2, 64, 32, [100, 50], 17)
    bounds, q = _dev(np.nan_to_num(_bounds_of(c), nan=0.0), np.float16), torch.zeros((2, 256), device="cuda")
    for bad in (bounds[:1], bounds.float(), bounds.cpu(), bounds.transpose(2, 3)):
        with pytest.raises(ValueError):
            ctx.paged_bounds(c.kv, c.pages, c.batch(), bad)
        with pytest.raises(ValueError):
            ctx.paged_attention_selected(c.kv, c.pages, bad, c.batch(), q, 4, 2)
    off = torch.zeros(bounds.numel() + 1, dtype=torch.float16, device="cuda")[1:]
    over = c.pages.view(torch.float16).view(-1)[:bounds.numel()].view(bounds.shape)
    for b in (off, over):
        with pytest.raises(KmoeError) as e:
            ctx.paged_bounds(c.kv, c.pages, c.batch(), b)
        assert e.value.status == -1
    call = lambda **k: ctx.paged_attention_selected(**{**dict(kv=c.kv, pages=c.pages, bounds=bounds, batch=c.batch(), q=q, n_head=4, n_select=2), **k})  # noqa: E731
    for bad in (dict(n_select=0), dict(n_select=-1), dict(n_first=2), dict(n_first=-1), dict(bounds=off), dict(out=q),
                dict(n_head=3, q=torch.zeros((2, 192), device="cuda"))):
        with pytest.raises(KmoeError) as e:
            call(**bad)
        assert e.value.status == -1, bad
    for bad in (dict(q=q.half()), dict(q=q[:1]), dict(out=q[:1])):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(KmoeError) as e:
        call(n_head=34, q=torch.zeros((2, 34 * 64), device="cuda"))
    assert e.value.status == -2
    many = PagedKV(F16, 8, 64, 32)
    p8, b8 = torch.zeros((1, many.page_bytes), dtype=torch.uint8, device="cuda"), torch.zeros((1, 8, 2, 64), dtype=torch.float16, device="cuda")
    for cols, ok in (((1 << 19) + 1, False), (1 << 19, True)):  # 2^22 columns by kv heads
        b = ctx.paged_batch(torch.full((1, cols), -1, dtype=torch.int32, device="cuda"), _dev([1 << 24], np.int32))
        if ok:
            assert not ctx.paged_attention_selected(many, p8, b8, b, torch.ones((1, 512), device="cuda"), 8, 3).any()
        else:
            with pytest.raises(KmoeError) as e:
                ctx.paged_attention_selected(many, p8, b8, b, torch.ones((1, 512), device="cuda"), 8, 3)
            assert e.value.status == -2
    wide = ctx.paged_batch(torch.zeros((1, (1 << 20) + 1), dtype=torch.int32, device="cuda"), _dev([1], np.int32))
    with pytest.raises(KmoeError) as e:
        call(batch=wide, q=q[:1].contiguous())
    assert e.value.status == -2
    torch.cuda.synchronize()
