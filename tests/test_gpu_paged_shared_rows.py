"""Attention over shared prefixes and selected pages of batches whose row_start reaches past the call's rows, or makes no
sense: nothing outside the call's rows is written, and rows that one sequence alone has are right."""
from types import SimpleNamespace

import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0
from tests.test_gpu_paged import _close, _dev, _reference, ctx  # noqa: F401  (ctx: a fixture)
from tests.test_gpu_paged_shared import _shared

pytestmark = pytest.mark.gpu
TYPES = [F16, Q8_0]
FORMS = ["shared", "selected"]


def _attend(c, form, batch, q, nh, start, pages, out):
    """Of `out`, longer than the call's rows: what the call leaves in all of it."""
    import torch

    dq, o = _dev(q.reshape(len(q), -1)), out[:len(q)]
    if form == "shared":
        c.ctx.paged_attention_shared(c.kv, c.pages, batch, c.ctx.paged_groups(_dev(start, np.int32), _dev(pages, np.int32), always=True), dq, nh, out=o)
    else:  # (all pages but one: as many as any row has)
        bounds = torch.zeros((c.pages.shape[0], c.kv.n_kv, 2, c.kv.head_dim), dtype=torch.float16, device="cuda")
        c.ctx.paged_attention_selected(c.kv, c.pages, c.ctx.paged_bounds(c.kv, c.pages, batch, bounds), batch, dq, nh, c.cols - 1, 0, out=o)
    torch.cuda.synchronize()
    return out.cpu().numpy()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rs,s_rows,rows", [([0, 1, 5, 7], 2, [1, 1, 0]), ([0, 1, 2 ** 31 - 2, 2 ** 31 - 1], 2, [1, 1, 0]),
                                            ([0, 2, 3, 90], 9, [2, 1, 6]), ([4, 4, 4, 4], 3, [0, 0, 0])])
def test_row_starts_past_the_calls_rows(ctx, t, form, rs, s_rows, rows):  # noqa: F811
    """One group over all three sequences, of which the last ones lie past the call's rows or reach past them."""
    nh, hd, lens, start, pages = 4, 64, [90, 100, 110], [0, 3], [2]
    c = _shared(ctx, t, 2, hd, 32, lens, start, pages, s_rows, extra_cols=1)
    q = np.random.default_rng(1).standard_normal((s_rows, nh, hd)).astype(np.float32)
    out = _dev(np.full((s_rows + 8, nh * hd), 7.0), np.float32)
    b = ctx.paged_batch(_dev(c.table), _dev(lens, np.int32), _dev(rs, np.int32), s_rows)
    got = _attend(c, form, b, q, nh, start, pages, out)
    n = sum(rows)
    assert (got[n:] == 7).all()
    if n:
        ref, tol, _ = _reference(c, q[:n], rows, nh)
        _close(got[:n], ref, tol * (1 + 8 / 64))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("nh", [2, 16])
def test_row_starts_that_make_no_sense(ctx, t, form, nh):  # noqa: F811
    hd, lens = 64, [70, 80, 90, 100, 75]
    for start, pages in (([0, 3, 5], [2, 1]), ([0, 5], [2]), ([1, 4], [1])):
        c = _shared(ctx, t, 1, hd, 32, lens, start, pages, nh, extra_cols=1)
        rs = _dev([5, 2, 9, -4, 3, 100], np.int32)  # rows none, 2 .. 7, none, 0 .. 2, 3 .. 7
        q = np.random.default_rng(2).standard_normal((8, nh, hd)).astype(np.float32)
        got = _attend(c, form, ctx.paged_batch(_dev(c.table), _dev(lens, np.int32), rs, 8), q, nh, start, pages, _dev(np.full((16, nh * hd), 7.0), np.float32))
        assert (got[8:] == 7).all()
        if form == "shared":  # rows 0 and 1 are one sequence's alone
            sub = SimpleNamespace(kv=c.kv, lens=[100], hk=[c.hk[3]], hv=[c.hv[3]])
            ref, tol, _ = _reference(sub, q[:3], [3], nh)
            _close(got[:2], ref[:2], tol[:2] * (1 + 8 / 64))
