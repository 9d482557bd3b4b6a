"""The paged key-value cache (kmoe_paged.hip, kmoe_paged_attn.hip) against plain
64-bit references: rows in and out, attention of decoding sequences, prompt
chunks and both, windows, pages that are missing, copies, captured calls."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0, F32, KmoeError, PagedKV

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0]


@pytest.fixture(scope="module")
def ctx():
    from kestrel_amd.kmoe import Context

    c = Context(0)
    yield c
    c.close()


def _dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def _held(t, x):
    """The values a cache of type t stands for after storing rows x [..., dims], 64 bits (Q8_0 by the format:
    f16 scale nearest to amax / 127, quants to the nearest, ties to even)."""
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float64)
    y = x.astype(np.float64).reshape(-1, 32)
    d = np.minimum((np.abs(y).max(1, keepdims=True).astype(np.float32) / np.float32(127)), 65504).astype(np.float16).astype(np.float64)
    q = np.clip(np.rint(np.divide(y, d, out=np.zeros_like(y), where=d > 0)), -127, 127)
    return (q * d).reshape(x.shape)


class Cache:
    """Sequences of given lengths stored row by row through the entry points, and their values in 64 bits."""

    def __init__(self, ctx, t, nkv, hd, page, lens, seed, extra_cols=0, scale=1.0, spare=3):
        import torch

        rng = np.random.default_rng(seed)
        self.kv, self.ctx, self.lens = PagedKV(t, nkv, hd, page), ctx, list(lens)
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + spare
        self.cols = max(need + [1]) + extra_cols
        ids, at = rng.permutation(n_pages), 0
        self.table = np.full((len(lens), self.cols), -1, np.int32)
        for b, m in enumerate(need):
            self.table[b, :m] = ids[at:at + m]
            at += m
        self.free = ids[at:].tolist()
        # stale bytes everywhere: NaNs in f16 elements and scales
        self.pages = torch.full((n_pages, self.kv.page_bytes), 0xff, dtype=torch.uint8, device="cuda")
        self.k, self.v = ([rng.standard_normal((n, nkv, hd)).astype(np.float32) * np.float32(scale) for n in lens] for _ in range(2))
        total = sum(lens)
        if total:
            rs = np.concatenate([[0], np.cumsum(lens)])
            b = ctx.paged_batch(_dev(self.table), _dev(lens, np.int32), _dev(rs, np.int32), total)
            ctx.paged_kv_store(self.kv, self.pages, b, _dev(np.concatenate(self.k).reshape(total, -1)),
                               _dev(np.concatenate(self.v).reshape(total, -1)))
        self.hk, self.hv = ([_held(t, x) for x in y] for y in (self.k, self.v))

    def batch(self, rows=None, lens=None, table=None, s_rows=None):
        lens = self.lens if lens is None else lens
        table = self.table if table is None else table
        rs = None if rows is None else _dev(np.concatenate([[0], np.cumsum(rows)]), np.int32)
        total = len(lens) if rows is None else sum(rows)
        return self.ctx.paged_batch(_dev(table), _dev(lens, np.int32), rs, total if s_rows is None else s_rows)


def _reference(c, q, rows, nh, window=0, sink=0, hidden=None):
    """softmax attention in 64 bits [S, nh, hd] and, per output element, a bound of what f32 arithmetic may be off."""
    nkv, hd = c.kv.n_kv, c.kv.head_dim
    out, tol, at = [], [], 0
    for b, n in enumerate(c.lens):
        r = 1 if rows is None else rows[b]
        for i in range(r):
            pos = n - r + i
            p = np.arange(n)
            see = p <= pos
            if window:
                see &= (p > pos - window) | (p < sink)
            if hidden is not None:
                see &= ~hidden[b]
            for h in range(nh):
                g = h // (nh // nkv)
                k, v, x = c.hk[b][see, g], c.hv[b][see, g], q[at, h].astype(np.float64)
                if not len(k):
                    out.append(np.zeros(hd))
                    tol.append(np.zeros(hd))
                    continue
                s = k @ x / np.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                out.append(w @ v)
                # a score: hd products summed in f32 chains of at most hd / 8 + 8 roundings of partial sums of at
                # most sum |q k|, and it enters the weight and the weights' sum; a weighted sum: chains of at
                # most n / 32 + 64 roundings
                e = 2 * (hd / 8 + 8) * (np.abs(k) @ np.abs(x) / np.sqrt(hd)).max() + n / 32 + 64
                tol.append(2.0 ** -24 * e * (w @ np.abs(v)))
            at += 1
    return np.array(out).reshape(at, nh, hd), np.array(tol).reshape(at, nh, hd), at


def _close(got, ref, tol, worst_score=6.0):
    got = got.reshape(ref.shape).astype(np.float64)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol + 1e-30).all(), np.abs(got - ref).max()
    # on the average the roundings add up like a few of a score's own: |score| 2^-23 each, and as much of its weight
    assert np.linalg.norm(got - ref) <= (4 + 2 * worst_score) * 2.0 ** -23 * max(np.linalg.norm(ref), 1e-30)


def _attend(c, q, nh, rows=None, **kw):
    import torch

    S = q.shape[0]
    o = c.ctx.paged_attention(c.kv, c.pages, c.batch(rows, s_rows=kw.pop("s_rows", None)), _dev(q.reshape(S, -1)), nh, **kw)
    torch.cuda.synchronize()
    return o.cpu().numpy()


# ------------------------------------------------------------ rows in and out

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nkv,hd,page,lens", [(1, 64, 32, [1]), (4, 128, 64, [37, 64, 65, 1, 200]), (3, 64, 256, [255, 256, 257]),
                                              (8, 128, 128, [300, 5])])
def test_rows_come_back_as_stored(ctx, t, nkv, hd, page, lens):
    c = Cache(ctx, t, nkv, hd, page, lens, 1, extra_cols=2, scale=3.0)
    k, v = ctx.paged_kv_read(c.kv, c.pages, c.batch(rows=lens))
    for got, want in ((k, c.hk), (v, c.hv)):
        want = np.concatenate(want).reshape(sum(lens), -1)
        assert np.array_equal(got.cpu().numpy(), want.astype(np.float16))


def test_q8_scales_and_ties(ctx):
    """Groups at the format's edges: zeros, one value, exact halves between two quants, scales below f16's normal
    range and past its largest, NaN and infinity (their group reads as NaN, no other)."""
    kv, page = PagedKV(Q8_0, 1, 64, 32), 32
    x = np.zeros((32, 64), np.float32)
    x[1, 3] = -5.0
    d = np.float32(np.float16(1.5))
    x[2, :32] = d * (np.arange(32) - 15.5)  # halves: scale 1.5 (amax 190.5 = 127 * 1.5)
    x[2, 31] = d * 127
    x[3, :32] = d * (np.arange(32) - 15.5) * (1 + 2.0 ** -20)
    x[3, 31] = d * 127
    x[4] = np.linspace(-3e-6, 3e-6, 64)
    x[5] = np.linspace(-9e6, 9e6, 64)
    x[6] = 1e-12
    x[7, 5], x[8, 40], x[9, 0] = np.nan, np.inf, -np.inf
    x[10:] = np.random.default_rng(0).standard_normal((22, 64)) * np.exp2(np.random.default_rng(1).integers(-18, 18, (22, 1)))
    import torch

    pages = torch.zeros((1, kv.page_bytes), dtype=torch.uint8, device="cuda")
    b = ctx.paged_batch(_dev([[0]], np.int32), _dev([32], np.int32), _dev([0, 32], np.int32), 32)
    ctx.paged_kv_store(kv, pages, b, _dev(x), _dev(-x))
    k, v = (a.cpu().numpy() for a in ctx.paged_kv_read(kv, pages, b))
    bad = np.zeros((32, 2), bool)
    bad[7, 0] = bad[8, 1] = bad[9, 0] = True
    bad = np.repeat(bad, 32, 1)
    clean = np.where(bad, 0, x).astype(np.float32)
    with np.errstate(over="ignore"):
        want = _held(Q8_0, clean).astype(np.float16)
    assert np.isnan(k[bad]).all() and np.isnan(v[bad]).all()
    assert np.array_equal(k[~bad], want[~bad]) and np.array_equal(v[~bad], -want[~bad])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,rd,neox", [(4, 2, 128, 128, True), (6, 3, 64, 32, False), (2, 2, 128, 64, True), (32, 8, 64, 64, False)])
def test_rope_store_takes_parts_of_a_projection(ctx, t, nh, nkv, hd, rd, neox):
    import torch

    rng = np.random.default_rng(nh)
    lens, rows, page = [1, 40, 3000, 64], [1, 7, 1, 64], 32
    c = Cache(ctx, t, nkv, hd, page, lens, 2)
    S = sum(rows)
    x = rng.standard_normal((S, (nh + 2 * nkv) * hd)).astype(np.float32)
    inv = (10000.0 ** (-np.arange(rd // 2) * 2.0 / rd)).astype(np.float32)
    xd, n, w = _dev(x), nh * hd, nkv * hd
    b = c.batch(rows)
    q = ctx.paged_rope_kv_store(c.kv, c.pages, b, xd[:, :n], xd[:, n:n + w], xd[:, n + w:], nh, rd, _dev(inv), neox)
    k, v = ctx.paged_kv_read(c.kv, c.pages, b)
    pos = np.concatenate([np.arange(m - r, m) for m, r in zip(lens, rows)])
    ang = (pos.astype(np.float32)[:, None] * inv).astype(np.float64)[:, None]

    def rot(y):
        y = y.reshape(S, -1, hd).astype(np.float64).copy()
        a, e = (y[..., :rd // 2].copy(), y[..., rd // 2:rd].copy()) if neox else (y[..., 0:rd:2].copy(), y[..., 1:rd:2].copy())
        i, j = (slice(0, rd // 2), slice(rd // 2, rd)) if neox else (slice(0, rd, 2), slice(1, rd, 2))
        y[..., i], y[..., j] = a * np.cos(ang) - e * np.sin(ang), a * np.sin(ang) + e * np.cos(ang)
        return y

    # two products, a sum and a sine and cosine within 2 ulp each: at most 8 half ulps of |x0| + |x1|
    lim = 8 * 2.0 ** -24 * np.abs(x).max() * 2
    assert np.abs(q.cpu().numpy().reshape(S, nh, hd) - rot(x[:, :n])).max() <= lim
    wk = rot(x[:, n:n + w])
    # one step of the cache's type may go the other way where the value lies on a border
    step = (np.abs(wk).reshape(S, nkv, -1, 32).max(-1, keepdims=True) / 127 * 1.01 + 0 * wk.reshape(S, nkv, -1, 32)).reshape(wk.shape) if t == Q8_0 else np.abs(wk) * 2.0 ** -10
    gk = k.cpu().numpy().reshape(S, nkv, hd).astype(np.float64)
    assert (np.abs(gk - wk) <= step / 2 + np.abs(wk) * 2.0 ** -11 + lim + 2.0 ** -25).all()
    assert np.array_equal(v.cpu().numpy(), _held(t, x[:, n + w:].reshape(S, nkv, hd)).reshape(S, w).astype(np.float16))
    # rows stored before are as they were
    rest = [m - r for m, r in zip(lens, rows)]
    k0, v0 = ctx.paged_kv_read(c.kv, c.pages, c.batch(rows=rest, lens=rest))
    assert np.array_equal(k0.cpu().numpy(), np.concatenate([h[:m] for h, m in zip(c.hk, rest)]).reshape(-1, w).astype(np.float16))
    # the same bits as the one-sequence entry points
    if t == F16:
        kc, vc = (torch.zeros((64, w), dtype=torch.int16, device="cuda") for _ in range(2))
        one = [xd[S - 64:, a:e].contiguous() for a, e in ((0, n), (n, n + w), (n + w, n + 2 * w))]
        q1 = ctx.rope_kv_store(*one, nh, nkv, hd, rd, 0, _dev(inv), neox, 64, kc, vc)
        assert torch.equal(q1.view(torch.int32), q[S - 64:].view(torch.int32))
        assert torch.equal(kc, k[S - 64:].view(torch.int16)) and torch.equal(vc, v[S - 64:].view(torch.int16))


@pytest.mark.parametrize("t", TYPES)
def test_rows_without_a_page_are_skipped(ctx, t):
    """Positions past the table, on missing pages and before the sequence's start write nothing, read as zeros, and
    rows behind the last sequence are left as they were."""
    import torch

    kv, page, w = PagedKV(t, 2, 64, 32), 32, 128
    table = np.array([[0, -1], [2, 99], [3, 4], [5, -7]], np.int32)  # of 8 pages
    lens, rows = [64, 40, 70, 3], [64, 10, 10, 5]
    pages = torch.full((8, kv.page_bytes), 0x11, dtype=torch.uint8, device="cuda")
    before = pages.clone()
    S = sum(rows) + 4
    x = np.random.default_rng(5).standard_normal((S, w)).astype(np.float32)
    b = ctx.paged_batch(_dev(table), _dev(lens, np.int32), _dev(np.concatenate([[0], np.cumsum(rows)]), np.int32), S)
    xd = _dev(x)
    ctx.paged_kv_store(kv, pages, b, xd, xd)
    inv = _dev(np.ones(32, np.float32))
    q = torch.full((S, w), 7.0, device="cuda")
    ctx.paged_rope_kv_store(kv, before.clone(), b, xd, xd, xd, 2, 64, inv, True, q_out=q)
    assert (q[-4:] == 7.0).all() and torch.isfinite(q).all() and not (q[:-4] == 7.0).any()
    k, v = torch.full((S, w), 7.0, dtype=torch.float16, device="cuda"), torch.full((S, w), 7.0, dtype=torch.float16, device="cuda")
    import ctypes as C

    ctx.check(ctx.lib.kmoe_paged_kv_read(ctx.h, C.byref(kv.desc(pages)), pages.data_ptr(), C.byref(b), k.data_ptr(), v.data_ptr()))
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
    seq = np.repeat(np.arange(4), rows)
    ok = np.array([0 <= p < 64 and 0 <= table[s, p // 32] < 8 for s, p in zip(seq, pos)])
    want = np.where(ok[:, None], _held(t, x[:-4].reshape(-1, 2, 64)).reshape(-1, w), 0).astype(np.float16)
    assert 20 < ok.sum() < len(ok) - 20
    assert np.array_equal(k[:-4].cpu().numpy(), want) and np.array_equal(v[:-4].cpu().numpy(), want)
    assert (k[-4:] == 7.0).all() and (v[-4:] == 7.0).all()
    for page_id in (1, 6, 7):  # named by nobody
        assert torch.equal(pages[page_id], before[page_id])


# ------------------------------------------------------------------ attention

HEADS = [(1, 1, 64), (4, 4, 128), (6, 2, 64), (5, 1, 128), (14, 2, 64), (16, 2, 128), (16, 1, 64), (32, 4, 128)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_one_row_per_sequence(ctx, t, nh, nkv, hd):
    """Decode: lengths on and around tile, page and work-group borders, and a long one that is split."""
    page = [32, 64, 128, 256][(nh + hd) % 4]
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 1000, 4001]
    c = Cache(ctx, t, nkv, hd, page, lens, nh + hd, extra_cols=1)
    q = np.random.default_rng(9).standard_normal((len(lens), nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, None, nh)
    _close(_attend(c, q, nh), ref, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page,n", [(4, 1, 128, 256, 20011), (2, 2, 64, 32, 9000), (1, 1, 128, 64, 1), (8, 1, 64, 128, 31)])
def test_one_sequence(ctx, t, nh, nkv, hd, page, n):
    c = Cache(ctx, t, nkv, hd, page, [n], n)
    q = np.random.default_rng(n).standard_normal((1, nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, None, nh)
    _close(_attend(c, q, nh), ref, tol)


@pytest.mark.parametrize("t,hd", [(F16, 64), (Q8_0, 64), (F16, 128)])
def test_one_head_over_a_long_context(ctx, t, hd):
    """A single kv head split over every work-group of the launch."""
    nh, n = 3, 300007
    c = Cache(ctx, t, 1, hd, 256, [n], 5)
    q = np.random.default_rng(n).standard_normal((1, nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, None, nh)
    _close(_attend(c, q, nh), ref, tol)
    rows = [9]
    q = np.random.default_rng(n).standard_normal((9, nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, rows, nh)
    _close(_attend(c, q, nh, rows), ref, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page,lens,rows", [
    (4, 2, 128, 64, [100], [100]), (8, 2, 64, 32, [333], [150]), (2, 2, 128, 128, [77, 200, 5], [77, 1, 5]),
    (16, 1, 64, 64, [40, 3, 90], [9, 3, 0]), (6, 2, 64, 32, [700, 33, 64, 1], [2, 17, 64, 1]), (3, 1, 128, 256, [600], [31]),
    (4, 4, 64, 32, [1, 1, 1], [1, 0, 1]), (16, 16, 128, 64, [65], [65]), (14, 2, 64, 64, [2100], [5]),
    (5, 1, 64, 32, [129, 700], [129, 300]), (16, 1, 128, 128, [1500], [257]), (1, 1, 128, 64, [513], [513])])
def test_chunks_and_mixed_batches(ctx, t, nh, nkv, hd, page, lens, rows):
    c = Cache(ctx, t, nkv, hd, page, lens, sum(lens))
    q = np.random.default_rng(1).standard_normal((sum(rows), nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, rows, nh)
    _close(_attend(c, q, nh, rows), ref, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (2, 0), (31, 4), (32, 0), (33, 1), (64, 32), (100, 37), (129, 300), (5000, 4)])
@pytest.mark.parametrize("rows", [None, [1, 20, 3, 70, 1, 40]])
def test_window_and_first_positions(ctx, t, window, sink, rows):
    nh, nkv, hd = (4, 2, 128) if window % 2 else (8, 2, 64)
    lens = [1, 64, 200, 97, 2500, 333]
    c = Cache(ctx, t, nkv, hd, 32, lens, window)
    q = np.random.default_rng(sink).standard_normal((sum(rows) if rows else 6, nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, rows, nh, window, sink)
    _close(_attend(c, q, nh, rows, window=window, n_sink=sink), ref, tol)
    # pages that no row sees are not read: their ids may be anything
    for b, n in enumerate(lens):
        r = rows[b] if rows else 1
        for col in range(c.cols):
            p = np.arange(32 * col, 32 * col + 32)
            if not ((p < n) & ((p > n - r - window) | (p < sink))).any():
                c.table[b, col] = -1 if col % 2 else 1 << 30
    _close(_attend(c, q, nh, rows, window=window, n_sink=sink), ref, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [None, [1, 0, 5, 40]])
def test_rows_that_see_nothing_give_zeros(ctx, t, rows):
    """Lengths of zero (a slot without a sequence), rows before the start, pages that are all missing; rows behind
    the last sequence stay."""
    import torch

    nh, nkv, hd = 4, 2, 64
    c = Cache(ctx, t, nkv, hd, 32, [50, 40, 96, 45], 3)
    c.table[2, :] = -1
    lens = [0, 40, 96, 30]
    S = 4 if rows is None else sum(rows)
    q = np.random.default_rng(1).standard_normal((S + 3, nh * hd)).astype(np.float32)
    out = torch.full((S + 3, nh * hd), 7.0, device="cuda")
    if rows is None:
        b, o, qd = c.batch(None, lens), out[:S], _dev(q[:S])
    else:
        b, o, qd = c.batch(rows, lens, s_rows=S + 3), out, _dev(q)
    ctx.paged_attention(c.kv, c.pages, b, qd, nh, out=o)
    got = out.cpu().numpy()
    assert (got[S:] == 7.0).all()
    if rows is None:
        assert (got[0] == 0).all() and (got[2] == 0).all() and np.isfinite(got[:S]).all() and (got[1] != 0).any()
    else:
        assert (got[:1] == 0).all() and (got[1:6] == 0).all()  # length 0; all pages missing
        assert (got[6:16] == 0).all() and (got[16:46] != 0).any(1).all()  # rows at -10 .. -1, then 0 .. 29


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [None, [1, 70, 3]])
def test_missing_pages_are_not_seen(ctx, t, rows):
    nh, nkv, hd, lens = 6, 2, 128, [400, 170, 65]
    c = Cache(ctx, t, nkv, hd, 32, lens, 8)
    hidden = []
    for b, n in enumerate(lens):
        h = np.zeros(n, bool)
        for col in ([1, 2, 7] if b == 0 else [0] if b == 1 else [1]):
            c.table[b, col] = [-1, 1 << 20, -(1 << 31)][col % 3]
            h[32 * col:32 * col + 32] = True
        hidden.append(h)
    q = np.random.default_rng(1).standard_normal((sum(rows) if rows else 3, nh, hd)).astype(np.float32)
    ref, tol, _ = _reference(c, q, rows, nh, hidden=hidden)
    _close(_attend(c, q, nh, rows), ref, tol)


def _spoil(c, b, p, what):
    """Position p of sequence b holds what (NaN or infinities) in K and V of every head, through the store."""
    n = c.kv.n_kv * c.kv.head_dim
    x = _dev(np.full((1, n), what, np.float32))
    bt = c.ctx.paged_batch(_dev(c.table[b:b + 1]), _dev([p + 1], np.int32))
    c.ctx.paged_kv_store(c.kv, c.pages, bt, x, x)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows", [None, [1, 33, 40]])
def test_what_a_row_does_not_see_cannot_spoil_it(ctx, t, what, rows):
    """NaNs and infinities behind the length, before the window, between the first positions and the window, and at
    the positions of later rows of the same tile."""
    nh, nkv, hd, window, sink = 4, 2, 128, 70, 3
    lens = [300, 200, 90]
    c = Cache(ctx, t, nkv, hd, 32, [n + 20 for n in lens], 11)
    c.lens, c.hk, c.hv = lens, [x[:n] for x, n in zip(c.hk, lens)], [x[:n] for x, n in zip(c.hv, lens)]
    for b, n in enumerate(lens):
        r = rows[b] if rows else 1
        for p in list(range(n, n + 20)) + [sink, sink + 1, n - r - window]:
            if p >= n or sink <= p <= n - r - window:
                _spoil(c, b, p, what)
    q = np.random.default_rng(1).standard_normal((sum(rows) if rows else 3, nh, hd)).astype(np.float32)
    ref, tol, S = _reference(c, q, rows, nh, window, sink)
    _close(_attend(c, q, nh, rows, window=window, n_sink=sink), ref, tol)
    if rows:  # a later row's own position: only the rows from there on see it
        _spoil(c, 1, 199, what)
        got = _attend(c, q, nh, rows, window=window, n_sink=sink).reshape(S, nh, hd)
        bad = 1 + 33 - 1
        assert not np.isfinite(got[bad]).any()
        keep = np.arange(S) != bad
        _close(got[keep], ref[keep], tol[keep])


@pytest.mark.parametrize("hd,rows", [(128, None), (64, None), (128, [40]), (64, [40])])
def test_infinities_that_a_row_sees(ctx, hd, rows):
    """f16 pages: an infinite V element reaches its own dim, as in plain arithmetic; a K row that scores -inf weighs
    nothing; an infinite q gives NaN."""
    nh, nkv, n = 4, 2, 150
    c = Cache(ctx, F16, nkv, hd, 32, [n], 4)
    r = 1 if rows is None else rows[0]
    k, v = c.k[0].copy(), c.v[0].copy()
    v[45, 0, 7], v[46, 1, 9], v[50, 0, 11] = np.inf, -np.inf, np.nan
    k[60, 0, 5] = -np.inf
    b = c.batch([n])
    c.ctx.paged_kv_store(c.kv, c.pages, b, _dev(k.reshape(n, -1)), _dev(v.reshape(n, -1)))
    q = np.random.default_rng(1).standard_normal((r, nh, hd)).astype(np.float32)
    q[:, :2, 5] = np.abs(q[:, :2, 5]) + 0.1  # kv head 0: every score of position 60 is -inf
    q[0, 3, 2] = np.inf
    c.hk, c.hv = [k.astype(np.float16).astype(np.float64)], [v.astype(np.float16).astype(np.float64)]
    with np.errstate(all="ignore"):
        ref, tol, S = _reference(c, q, rows, nh)
    got = _attend(c, q, nh, rows).reshape(ref.shape)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(np.isposinf(got), np.isposinf(ref)) and np.array_equal(np.isneginf(got), np.isneginf(ref))
    f = np.isfinite(ref)
    assert np.isposinf(ref).any() and np.isneginf(ref).any() and 0.7 < f.mean() < 1
    _close(got[f], ref[f], tol[f])


# the smallest bits: a first position with a zero value that takes all but e^-20 of the weight, and a q element 2^24
# above the others whose K is zero (f16 holds neither's rest in one piece); f32's bits are kept
@pytest.mark.parametrize("kind", ["sink", "outlier"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [None, [37]])
def test_small_weights_and_elements_keep_their_bits(ctx, kind, hd, rows):
    rng = np.random.default_rng(hd)
    nh, nkv, n = 4, 2, 160
    r = 1 if rows is None else rows[0]
    c = Cache(ctx, F16, nkv, hd, 32, [n], 4)
    q = rng.standard_normal((r, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float16).astype(np.float32) for _ in range(2))
    if kind == "sink":
        q[:, :, 0] = 8.0
        k[:, :, 0] = 0.0
        k[0] = 0.0
        k[0, :, 0] = 20 * np.sqrt(hd) / 8.0
        v[0] = 0.0
    else:
        q[:, :, 3] = 2.0 ** 24
        k[:, :, 3] = 0.0
    ctx.paged_kv_store(c.kv, c.pages, c.batch([n]), _dev(k.reshape(n, -1)), _dev(v.reshape(n, -1)))
    c.hk, c.hv = [k.astype(np.float16).astype(np.float64)], [v.astype(np.float64)]
    ref, _, S = _reference(c, q, rows, nh)
    got = _attend(c, q, nh, rows).reshape(S, nh, hd)
    for s in range(S):
        for h in range(nh):
            # an f32 score is off by up to |score| 2^-23, and as much of its weight (20 at the sink)
            assert np.linalg.norm(got[s, h] - ref[s, h]) <= (3e-6 if kind == "sink" else 1.5e-6) * np.linalg.norm(ref[s, h])


# Q8_0: a weight is off by up to 2^-36 of the largest besides its own 2^-23, an element of q by 2^-40 of the row's
# largest
@pytest.mark.parametrize("kind", ["sink", "outlier"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [None, [37]])
def test_q8_small_weights_and_elements(ctx, kind, hd, rows):
    rng = np.random.default_rng(hd + 1)
    nh, nkv, n = 4, 2, 160
    r = 1 if rows is None else rows[0]
    c = Cache(ctx, Q8_0, nkv, hd, 32, [n], 4)
    q = rng.standard_normal((r, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
    if kind == "sink":
        q[:, :, 0] = 8.0
        k[:, :, 0] = 0.0
        k[0] = 0.0
        k[0, :, 0] = 10 * np.sqrt(hd) / 8.0
        v[0] = 0.0
    else:
        q[:, :, 3] = 2.0 ** 16
        k[:, :, 3] = 0.0
    ctx.paged_kv_store(c.kv, c.pages, c.batch([n]), _dev(k.reshape(n, -1)), _dev(v.reshape(n, -1)))
    c.hk, c.hv = [_held(Q8_0, k)], [_held(Q8_0, v)]  # (the rows that paged_kv_read gives are rounded to f16)
    ref, tol, S = _reference(c, q, rows, nh)
    got = _attend(c, q, nh, rows).reshape(S, nh, hd)
    # sink: n weights, the largest 1, values up to 5. outlier: a score is off by that much of hd elements with |k| up
    # to 5, and so, in units of the weights (1 together), is each weight, with values up to 5
    more = n * 2.0 ** -36 * 5 if kind == "sink" else 2.0 ** 16 * 2.0 ** -40 * hd * 5 / np.sqrt(hd) * 5
    assert (np.abs(got - ref) <= tol + more).all()


@pytest.mark.parametrize("t", TYPES)
def test_scores_of_any_size(ctx, t):
    """Rows of very different size, from almost even weights to a single position's."""
    nh, nkv, hd = 8, 2, 128
    lens = [100 + 37 * i for i in range(12)]
    c = Cache(ctx, t, nkv, hd, 64, lens, 2, scale=2.0)
    q = np.random.default_rng(3).standard_normal((12, nh, hd)).astype(np.float32)
    q *= np.exp2(np.arange(12) - 9.0)[:, None, None].astype(np.float32)
    ref, tol, _ = _reference(c, q, None, nh)
    got = _attend(c, q, nh).reshape(ref.shape)
    assert (np.abs(got - ref) <= tol).all()


def test_the_same_call_gives_the_same_bits(ctx):
    lens = [5000, 3, 700, 64, 1]
    c = Cache(ctx, F16, 2, 128, 64, lens, 2)
    q = np.random.default_rng(3).standard_normal((5, 16, 128)).astype(np.float32)
    got = [_attend(c, q, 16) for _ in range(4)]
    assert all(np.array_equal(g.view(np.uint32), got[0].view(np.uint32)) for g in got)


def test_matches_the_one_sequence_entry_points(ctx):
    """The contiguous cache's attention on the same rows, decode and prompt."""
    import torch

    nh, nkv, hd, n = 16, 4, 128, 700
    c = Cache(ctx, F16, nkv, hd, 64, [n], 6)
    kc, vc = (_dev(np.ascontiguousarray(x[0].astype(np.float16).reshape(n, -1)).view(np.int16)) for x in (c.k, c.v))
    for r in (1, 40):
        q = np.random.default_rng(r).standard_normal((r, nh * hd)).astype(np.float32)
        a = ctx.attention(_dev(q), kc, vc, nh, nkv, hd, n - r, n).cpu().numpy()
        b = ctx.paged_attention(c.kv, c.pages, c.batch([r]), _dev(q), nh).cpu().numpy()
        assert np.linalg.norm(a - b) <= 3e-6 * np.linalg.norm(a)  # twice the bound of either
    torch.cuda.synchronize()


# -------------------------------------------------------------- pages copied

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layers,n_pages,n", [(1, 2, 1), (3, 40, 13), (2, 700, 300), (5, 6, 3)])
def test_copies(ctx, t, layers, n_pages, n):
    import torch

    kv = PagedKV(t, 3, 64, 32)
    g = torch.Generator(device="cuda").manual_seed(n)
    pages = torch.randint(0, 256, (layers, n_pages, kv.page_bytes), dtype=torch.uint8, device="cuda", generator=g)
    want = pages.clone()
    ids = np.random.default_rng(n).permutation(n_pages)
    dst = ids[:n].tolist()
    src = np.random.default_rng(n + 1).choice(ids[n:], n).tolist()  # one page onto several, too
    ctx.pages_copy(kv, pages, src, dst, n_layer=layers)
    want[:, dst] = want[:, src]
    assert torch.equal(pages, want)
    ctx.pages_copy(kv, pages, [], [], n_layer=layers)
    assert torch.equal(pages, want)


def test_copies_are_refused(ctx):
    import torch

    kv = PagedKV(F16, 1, 64, 32)
    pages = torch.zeros((2, 4, kv.page_bytes), dtype=torch.uint8, device="cuda")
    for s, d in (([0], [4]), ([4], [0]), ([-1], [0]), ([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(KmoeError) as e:
            ctx.pages_copy(kv, pages, s, d, n_layer=2)
        assert e.value.status == -1
    with pytest.raises(ValueError):
        ctx.pages_copy(kv, pages, [0, 1], [2], n_layer=2)


# ------------------------------------------------ streams, graphs, large pools

def test_captured_step_follows_its_lengths(ctx):
    """Store and attention captured once, replayed with other rows, lengths and tables; eager calls between the
    replays give the same bits."""
    import torch

    nh, nkv, hd, n_seq = 8, 2, 128, 5
    c = Cache(ctx, F16, nkv, hd, 32, [3000, 1500, 900, 64, 300], 7, extra_cols=2)
    g = np.random.default_rng(0)
    qkv = torch.zeros((n_seq, (nh + 2 * nkv) * hd), device="cuda")
    lens, table = torch.zeros(n_seq, dtype=torch.int32, device="cuda"), _dev(c.table)
    inv = _dev((10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)).astype(np.float32))
    b = ctx.paged_batch(table, lens)
    n, w = nh * hd, nkv * hd
    q, o = torch.zeros((n_seq, n), device="cuda"), torch.zeros((n_seq, n), device="cuda")

    def step(pages):
        ctx.paged_rope_kv_store(c.kv, pages, b, qkv[:, :n], qkv[:, n:n + w], qkv[:, n + w:], nh, hd, inv, True, q_out=q)
        ctx.paged_attention(c.kv, pages, b, q, nh, window=2048, n_sink=4, out=o)

    step(c.pages)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ctx.set_stream(torch.cuda.current_stream())
            step(c.pages)
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i, ln in enumerate(([2990, 1, 900, 64, 17], [1, 1, 1, 1, 1], [2999, 1499, 0, 33, 300], [40, 1400, 3, 2, 1])):
        x = _dev(g.standard_normal(qkv.shape).astype(np.float32))
        lens.copy_(_dev(ln, np.int32))
        qkv.copy_(x)
        keep = c.pages.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, pages = o.clone(), c.pages.clone()
        o.zero_()
        c.pages.copy_(keep)
        step(c.pages)
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int32), o.view(torch.int32)) and torch.equal(pages, c.pages), i
        assert torch.isfinite(got).all()


def test_capture_before_any_eager_call():
    """A context whose first attention call is a captured one."""
    import torch

    from kestrel_amd.kmoe import Context

    ctx = Context(0)
    c = Cache(ctx, F16, 2, 64, 32, [4000], 7)
    qd = _dev(np.random.default_rng(1).standard_normal((1, 4 * 64)).astype(np.float32))
    o = torch.zeros((1, 4 * 64), device="cuda")
    b = c.batch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ctx.set_stream(torch.cuda.current_stream())
            ctx.paged_attention(c.kv, c.pages, b, qd, 4, out=o)
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    want = ctx.paged_attention(c.kv, c.pages, b, qd, 4)
    for _ in range(3):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
    del graph
    ctx.close()


def test_calls_on_alternating_streams(ctx):
    """Split calls on two streams in turn, nothing waited for between: each gives its own result."""
    import torch

    cs = [Cache(ctx, F16, 2, 128, 64, [6000, 5000], s) for s in (1, 2)]
    qs = [_dev(np.random.default_rng(s).standard_normal((2, 8 * 128)).astype(np.float32)) for s in (1, 2)]
    bs = [c.batch() for c in cs]
    want = [ctx.paged_attention(c.kv, c.pages, b, q, 8) for c, b, q in zip(cs, bs, qs)]
    torch.cuda.synchronize()
    main, streams = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(want[0]) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    try:
        for i in range(20):
            for j in range(2):
                ctx.set_stream(streams[j])
                ctx.paged_attention(cs[j].kv, cs[j].pages, bs[j], qs[j], 8, out=outs[j][i])
    finally:
        ctx.set_stream(main)
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, want[j]) for o in outs[j])


@pytest.mark.parametrize("t", TYPES)
def test_pages_past_four_gigabytes(ctx, t):
    """A pool whose offsets pass 32 bits, bytes and elements."""
    import torch

    kv = PagedKV(t, 8, 128, 256)
    n_pages = (9 << 30) // kv.page_bytes + 3
    pages = torch.empty((n_pages, kv.page_bytes), dtype=torch.uint8, device="cuda")
    ids = [n_pages - 1, 0, n_pages // 2 + 1]
    n, nh = 700, 16
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((n, 8, 128)).astype(np.float32) for _ in range(2))
    b = ctx.paged_batch(_dev([ids], np.int32), _dev([n], np.int32), _dev([0, n], np.int32), n)
    ctx.paged_kv_store(kv, pages, b, _dev(k.reshape(n, -1)), _dev(v.reshape(n, -1)))
    gk, _ = ctx.paged_kv_read(kv, pages, b)
    assert np.array_equal(gk.cpu().numpy(), _held(t, k).reshape(n, -1).astype(np.float16))
    ctx.pages_copy(kv, pages, [n_pages - 1, 0], [n_pages - 2, 1])

    class One:
        pass

    c = One()
    c.kv, c.lens, c.hk, c.hv = kv, [n], [_held(t, k)], [_held(t, v)]
    q = rng.standard_normal((1, nh, 128)).astype(np.float32)
    ref, tol, _ = _reference(c, q, None, nh)
    for row in (ids, [n_pages - 2, 1, ids[2]]):
        b = ctx.paged_batch(_dev([row], np.int32), _dev([n], np.int32))
        _close(ctx.paged_attention(kv, pages, b, _dev(q.reshape(1, -1)), nh).cpu().numpy(), ref, tol)


# ------------------------------------------------------------------- refusals

def test_refusals(ctx):
    import ctypes as C

    import torch

    kv = PagedKV(F16, 2, 64, 32)
    pages = torch.zeros((4, kv.page_bytes), dtype=torch.uint8, device="cuda")
    table, lens = _dev([[0, 1]], np.int32), _dev([40], np.int32)
    x, q, w = torch.zeros((1, 128), device="cuda"), torch.zeros((1, 256), device="cuda"), 128
    out = torch.zeros_like(q)
    b = ctx.paged_batch(table, lens)
    inv = torch.ones(32, device="cuda")
    L, by = ctx.lib, C.byref

    def att(d=None, bt=b, p=pages.data_ptr(), qp=q.data_ptr(), nh=4, win=0, sink=0, o=out.data_ptr()):
        return L.kmoe_paged_attention(ctx.h, by(d or kv.desc(pages)), p, by(bt), qp, nh, win, sink, o)

    def batch(**kw):
        from kestrel_amd.kmoe import PagedBatch

        v = dict(n_seq=1, table_cols=2, s_rows=1, row_start=None, seq_len=lens.data_ptr(), table=table.data_ptr())
        v.update(kw)
        return PagedBatch(**v)

    from kestrel_amd.kmoe import PagedDesc as D

    INV, UNS = -1, -2
    for want, rc in [
            (0, att()), (INV, att(nh=3)), (INV, att(nh=0)), (UNS, att(nh=34)), (INV, att(win=-1)), (INV, att(sink=-1)),
            (INV, att(p=None)), (INV, att(p=pages.data_ptr() + 4)), (INV, att(qp=None)), (INV, att(o=None)), (INV, att(o=q.data_ptr())), (INV, att(o=q.data_ptr() + 4)),
            (UNS, att(D(F32, 2, 64, 32, 4))), (UNS, att(D(F16, 2, 96, 32, 4))), (UNS, att(D(F16, 2, 64, 16, 4))),
            (UNS, att(D(F16, 2, 64, 48, 4))), (INV, att(D(F16, 0, 64, 32, 4))), (INV, att(D(F16, 2, 64, 32, 0))),
            (INV, att(D(F16, 2, 64, 32, 1 << 31))), (INV, att(bt=batch(n_seq=-1))), (INV, att(bt=batch(n_seq=4097, s_rows=4097))),
            (INV, att(bt=batch(s_rows=2))), (INV, att(bt=batch(s_rows=-1, row_start=lens.data_ptr()))),
            (INV, att(bt=batch(seq_len=None))), (INV, att(bt=batch(table=None))), (INV, att(bt=batch(table_cols=-1))), (INV, att(bt=batch(table_cols=(1 << 25) + 1))),
            (INV, att(bt=batch(s_rows=(1 << 22) + 1, row_start=lens.data_ptr()))),
            (0, att(bt=batch(n_seq=0, s_rows=0, seq_len=None, table=None), p=None, qp=None, o=None)),
            (INV, L.kmoe_paged_kv_store(ctx.h, by(kv.desc(pages)), pages.data_ptr(), by(b), x.data_ptr(), w - 1, x.data_ptr(), w)),
            (INV, L.kmoe_paged_kv_store(ctx.h, by(kv.desc(pages)), pages.data_ptr(), by(b), None, w, x.data_ptr(), w)),
            (INV, L.kmoe_paged_kv_read(ctx.h, by(kv.desc(pages)), pages.data_ptr(), by(b), None, None)),
            (INV, L.kmoe_paged_attention(ctx.h, None, pages.data_ptr(), by(b), q.data_ptr(), 4, 0, 0, q.data_ptr())),
            (INV, L.kmoe_paged_attention(ctx.h, by(kv.desc(pages)), pages.data_ptr(), None, q.data_ptr(), 4, 0, 0, q.data_ptr())),
            (INV, L.kmoe_paged_attention(None, by(kv.desc(pages)), pages.data_ptr(), by(b), q.data_ptr(), 4, 0, 0, q.data_ptr()))]:
        assert rc == want
    for rd in (0, 3, 66, -2):
        with pytest.raises((KmoeError, ValueError)):
            ctx.paged_rope_kv_store(kv, pages, b, q, x, x, 4, rd, inv[:max(0, rd // 2)], True)
    for bad in (lambda: ctx.paged_attention(kv, pages, b, q.half(), 4), lambda: ctx.paged_attention(kv, pages, b, q.cpu(), 4),
                lambda: ctx.paged_attention(kv, pages, b, q, 2), lambda: ctx.paged_batch(table.long(), lens),
                lambda: ctx.paged_batch(table, lens, lens, 1), lambda: ctx.paged_batch(table, lens, _dev([0, 1], np.int32)),
                lambda: ctx.paged_kv_store(kv, pages, b, x[:, ::2], x), lambda: ctx.paged_attention(kv, pages.cpu(), b, q, 4),
                lambda: ctx.paged_kv_read(kv, pages[::2], b), lambda: ctx.paged_kv_store(kv, pages.cpu(), b, x, x),
                lambda: ctx.pages_copy(kv, pages.cpu(), [0], [1])):
        with pytest.raises(ValueError):
            bad()
