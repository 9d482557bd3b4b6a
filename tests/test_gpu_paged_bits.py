"""The smallest bits of the paged attention on Q8_0 pages: as f32 arithmetic's, like those on F16 pages."""
import numpy as np
import pytest

from kestrel_amd.kmoe import Q8_0
from tests.test_gpu_paged import Cache, _attend, _dev, _held, _reference, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


# a first position with a zero value that takes all but e^-20 of the weight, and a q element 2^24 above the others whose
# K is zero: f16 holds neither's rest in one piece
@pytest.mark.parametrize("kind", ["sink", "outlier"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [None, [37]])
def test_small_weights_and_elements_on_q8_pages(ctx, kind, hd, rows):  # noqa: F811
    rng = np.random.default_rng(hd + 7)
    nh, nkv, n = 4, 2, 160
    r = 1 if rows is None else rows[0]
    c = Cache(ctx, Q8_0, nkv, hd, 32, [n], 4)
    q = rng.standard_normal((r, nh, hd)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
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
    c.hk, c.hv = [_held(Q8_0, k)], [_held(Q8_0, v)]
    ref, _, S = _reference(c, q, rows, nh)
    got = _attend(c, q, nh, rows).reshape(S, nh, hd)
    # an f32 score is off by up to |score| 2^-23, and as much of its weight (20 at the sink): 3e-6, 1.5e-6. The product
    # of what the first f16 piece leaves of a weight (2^-36 of the largest) and of a value (2^-11 of it) is left out:
    # 2^-18 of a weight of e^-20 at most
    tol = 3e-6 + 2.0 ** -18 if kind == "sink" else 1.5e-6
    for s in range(S):
        for h in range(nh):
            assert np.linalg.norm(got[s, h] - ref[s, h]) <= tol * np.linalg.norm(ref[s, h])
