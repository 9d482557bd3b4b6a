"""Rows that the paged attention forms again in plain f32: those whose result is not finite and those without a score
above -inf."""
from types import SimpleNamespace

import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0
from tests.test_gpu_paged import Cache, _attend, _close, _dev, _reference, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,rows,window,sink,low", [
    (700, None, 100, 1, [0]),                   # the first position alone in its 256, the window further on
    (600, None, 345, 0, [255]),                 # the window begins at the last position of a block
    (600, None, 0, 0, range(256)),              # a whole block
    (900, [60], 0, 0, range(512)),
    (900, [60], 200, 3, [0, 1, 2, *range(641, 768)]),
])
def test_scores_of_minus_infinity_before_finite_ones(ctx, hd, n, rows, window, sink, low):  # noqa: F811
    """Positions that score -inf weigh nothing, wherever they lie: as if they were not seen."""
    nh, nkv = 8, 2
    c = Cache(ctx, F16, nkv, hd, 32, [n], 4)
    r = 1 if rows is None else rows[0]
    k = c.k[0].copy()
    low = np.isin(np.arange(n), list(low))
    k[low, :, 5] = -np.inf
    ctx.paged_kv_store(c.kv, c.pages, c.batch([n]), _dev(k.reshape(n, -1)), _dev(c.v[0].reshape(n, -1)))
    q = np.random.default_rng(1).standard_normal((r, nh, hd)).astype(np.float32)
    q[:, :, 5] = np.abs(q[:, :, 5]) + 0.1
    ref, tol, _ = _reference(c, q, rows, nh, window, sink, hidden=[low])
    _close(_attend(c, q, nh, rows, window=window, n_sink=sink), ref, tol)


@pytest.mark.parametrize("rows", [None, [40]])
def test_scores_of_minus_infinity_alone(ctx, rows):  # noqa: F811
    """The softmax of a row whose every visible score is -inf is not defined: NaN, in that row only."""
    nh, nkv, hd, n = 8, 2, 128, 700
    c = Cache(ctx, F16, nkv, hd, 32, [n], 4)
    r = 1 if rows is None else rows[0]
    k = c.k[0].copy()
    k[:n, 0, 5] = -np.inf
    ctx.paged_kv_store(c.kv, c.pages, c.batch([n]), _dev(k.reshape(n, -1)), _dev(c.v[0].reshape(n, -1)))
    q = np.random.default_rng(1).standard_normal((r, nh, hd)).astype(np.float32)
    q[:, :, 5] = np.abs(q[:, :, 5]) + 0.1
    got = _attend(c, q, nh, rows).reshape(r, nh, hd)
    assert np.isnan(got[:, :4]).all()
    ref, tol, _ = _reference(c, q, rows, nh)
    _close(got[:, 4:], ref[:, 4:], tol[:, 4:])


@pytest.mark.parametrize("t", [F16, Q8_0])
@pytest.mark.parametrize("nh,rows", [(4, None), (16, [5])])
@pytest.mark.parametrize("window,sink", [(0, 0), (50, 4), (2 ** 31 - 40, 0)])
def test_lengths_far_past_the_table(ctx, t, nh, rows, window, sink):  # noqa: F811
    """A slot with a stale length near 2^31: without pages its rows are zeros; with a NaN in the one page that it has,
    the rows that see it are NaN and the others what their own positions give. Many missing pages are passed over."""
    import torch

    nkv, hd = 1, 64
    c = Cache(ctx, t, nkv, hd, 32, [96], 11)
    S = 1 if rows is None else rows[0]
    q = np.random.default_rng(11).standard_normal((S, nh, hd)).astype(np.float32)
    for cols in (1, 3, 5000):
        table = np.full((1, cols), -1, np.int32)
        b = c.batch(rows, lens=[2 ** 31 - 1], table=table)
        out = torch.full((S, nh * hd), 3.0, device="cuda")
        ctx.paged_attention(c.kv, c.pages, b, _dev(q.reshape(S, -1)), nh, window=window, n_sink=sink, out=out)
        torch.cuda.synchronize()
        assert not out.any()
    k = c.k[0].copy()
    k[2] = np.nan
    ctx.paged_kv_store(c.kv, c.pages, c.batch([96]), _dev(k.reshape(96, -1)), _dev(c.v[0].reshape(96, -1)))
    table = np.full((1, 5000), -1, np.int32)
    table[0, 0] = c.table[0, 0]
    table[0, 4999] = c.table[0, 1]
    b = c.batch(rows, lens=[2 ** 31 - 1], table=table)
    out = ctx.paged_attention(c.kv, c.pages, b, _dev(q.reshape(S, -1)), nh, window=window, n_sink=sink).cpu().numpy()
    if not window or sink > 2:
        assert np.isnan(out).all()
    else:  # position 39 + row and on: the second of the two pages
        held = SimpleNamespace(kv=c.kv, lens=[32], hk=[c.hk[0][32:64]], hv=[c.hv[0][32:64]])
        for i in range(S):
            ref, tol, _ = _reference(held, q[i:i + 1], None, nh)
            _close(out[i:i + 1], ref, tol)
