"""Which pages are chosen, told from the values alone: keys that score nothing, values of each page's own."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0
from tests.test_gpu_paged import Cache, _close, _dev, _held, ctx  # noqa: F401  (ctx: a fixture)
from tests.test_gpu_paged_selected import _attend, _bounds_of, _reference_selected, _select

pytestmark = pytest.mark.gpu


def _refill(c, b, k, v):
    """Other keys and values for all positions of sequence b."""
    n = c.lens[b]
    batch = c.ctx.paged_batch(_dev(c.table[b:b + 1]), _dev([n], np.int32), _dev([0, n], np.int32), n)
    c.ctx.paged_kv_store(c.kv, c.pages, batch, _dev(k.reshape(n, -1)), _dev(v.reshape(n, -1)))
    c.hk[b], c.hv[b] = _held(c.kv.type, k), _held(c.kv.type, v)


@pytest.mark.parametrize("t", [F16, Q8_0])
@pytest.mark.parametrize("scale", [1.0, 1.0e-30, 1.0e30, -1.0e30, 3.0e38])
def test_scores_of_any_size(ctx, t, scale):  # noqa: F811
    """Bounds of both signs over forty powers of two, equal ones among them, times q of any size: products up to 2^142 are
    told apart."""
    rng = np.random.default_rng(13)
    n_pages = 700
    c = Cache(ctx, t, 1, 64, 32, [32 * n_pages], 13)
    v = np.repeat(rng.standard_normal((n_pages, 1, 64)), 32, axis=0).astype(np.float32)
    _refill(c, 0, np.zeros((32 * n_pages, 1, 64), np.float32), v)
    bounds = np.zeros((c.pages.shape[0], 1, 2, 64), np.float16)
    e = rng.choice(np.concatenate([2.0 ** np.arange(-24, 15), -2.0 ** np.arange(-24, 15), [0.0]]), n_pages)
    bounds[c.table[0], 0, :, 0] = e[:, None]
    q = np.zeros((1, 1, 64), np.float32)
    q[0, 0, 0] = scale
    seen = []
    for n_select in (2, 100, 350, 600, 699):
        hidden = _select(c, q, None, 1, n_select, 0, bounds)
        assert (~hidden[0]).sum() == 32 * n_select
        ref, tol = _reference_selected(c, q, None, 1, hidden)
        _close(_attend(c, q, 1, n_select, bounds=_dev(bounds, np.float16)), ref, tol)
        seen.append(ref)
    assert all(np.abs(a - b).max() > 1e-3 for a, b in zip(seen, seen[1:]))


@pytest.mark.parametrize("rows", [1, 40])
def test_what_is_not_finite_on_pages_that_are_not_chosen(ctx, rows):  # noqa: F811
    """Keys of NaN, of -inf, and values of both, on two pages whose other keys no row wants."""
    rng = np.random.default_rng(14)
    n = 330
    c = Cache(ctx, F16, 1, 64, 32, [n], 14)
    k, v = rng.standard_normal((n, 1, 64)).astype(np.float32), rng.standard_normal((n, 1, 64)).astype(np.float32)
    k[2 * 32:3 * 32] = k[5 * 32:6 * 32] = -4
    k[2 * 32 + 5, 0, 7] = -np.inf
    k[5 * 32 + 1] = np.nan
    v[2 * 32 + 9], v[5 * 32 + 30] = np.inf, np.nan
    _refill(c, 0, k, v)
    q = np.abs(rng.standard_normal((rows, 2, 64))).astype(np.float32)
    for n_select in (2, 4):
        hidden = _select(c, q, [rows], 2, n_select, 0, _bounds_of(c))
        assert hidden[0][:, 0, 2 * 32:3 * 32].all() and hidden[0][:, 0, 5 * 32:6 * 32].all()
        ref, tol = _reference_selected(c, q, [rows], 2, hidden)
        _close(_attend(c, q, 2, n_select, rows=[rows]), ref, tol)
