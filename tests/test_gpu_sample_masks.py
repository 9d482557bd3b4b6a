"""kmoe_sample where the first or the last chunks of a row hold nothing that can be drawn: weights of less than half of
2^-43 of the largest one's."""
import numpy as np
import pytest

from tests.test_gpu_sample import _check, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu
# below 0 and NaN count as 0, from 1 on the last token of any weight is drawn
U = np.array([0.0, -1.0, np.nan, 2.0 ** -126, 0.5, 1.0 - 2.0 ** -24, 1.0, np.inf], np.float32)


@pytest.mark.parametrize("low", [-1.0e9, -35.0, -30.6, -np.inf])
@pytest.mark.parametrize("n", [8000, 8193, 32000, 151936])
def test_masked_tokens_are_not_drawn(ctx, n, low):  # noqa: F811
    """e^-30.6 is 0.45 of 2^-43. Some visible tokens in the middle of a row: in one chunk, and across one's end."""
    rng = np.random.default_rng(n)
    for first, k in ((n // 2 // 1024 * 1024 + 100, 50), (n // 2 // 1024 * 1024 - 3, 6), (0, 1), (n - 1, 1)):
        x = np.full((U.size, n), low, np.float32)
        x[:, first:first + k] = rng.standard_normal((U.size, k)) * 0.1
        x[:, first + k // 2] = 0.5
        top = x.max(1, keepdims=True)
        x = np.where(x > -20, x - top, x).astype(np.float32)
        for how in (dict(), dict(temp=0.9), dict(p=0.9), dict(k=30)):
            ids = _check(ctx, x, U, **how)
            assert ((ids >= first) & (ids < first + k)).all()


@pytest.mark.parametrize("n", [32000, 151936])
def test_a_chunk_with_one_token_that_can_be_drawn(ctx, n):  # noqa: F811
    """One token of 0.6 of 2^-43 in an early and in a late chunk, all others at 0.4 of it: u = 0 and 1 find those."""
    x = np.full((U.size, n), -30.72, np.float32)
    x[:, n // 2] = 0.0
    x[:, [5000, n - 700]] = -30.316
    ids = _check(ctx, x, U)
    assert ids.tolist() == [5000] * 4 + [n // 2] * 2 + [n - 700] * 2


@pytest.mark.parametrize("n", [9000, 32000, 151936])
def test_the_last_token_where_sums_are_rounded_down(ctx, n):  # noqa: F811
    """The last tokens weigh 0.556 of 2^-43 each, which counts as 2^-43: u = 1 finds the last one all the same."""
    x = np.full((U.size, n), -np.inf, np.float32)
    x[:, n // 2] = 0.0
    x[:, n - 300:n - 20] = -30.392
    ids = _check(ctx, x, U)
    assert ids.tolist() == [n // 2] * 6 + [n - 21] * 2
