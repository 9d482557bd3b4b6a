"""What a sampled decode makes of its random numbers and settings (Decoder._sampling), on the CPU."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from kestrel_amd.decoder import Decoder

SETTINGS = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
BELOW = float(np.nextafter(np.float32(1), np.float32(0)))


def _u(u, rows=1, n=None):
    x = Decoder._sampling(SimpleNamespace(torch=torch, dev=torch.device("cpu")), {}, rows, u, len(u) if n is None else n, **SETTINGS)
    assert x.dtype is torch.float32 and x.is_contiguous()
    return x


@pytest.mark.parametrize("make", [list, np.array, lambda u: torch.tensor(u, dtype=torch.float64)])
def test_numbers_below_one_stay_below_one(make):
    """64-bit numbers next to 1, which 32 bits round to 1: there the last kept token is drawn."""
    u = [1 - 2.0 ** -53, 1 - 1e-9, 1 - 2.0 ** -25, 1 - 2.0 ** -24, 0.999999, 0.0, 1e-300]
    x = _u(make(u))
    assert x[:4, 0].tolist() == [BELOW] * 4 and x[4:, 0].tolist() == np.float32(u[4:]).tolist()


def test_numbers_past_their_range_are_the_callers():
    x = _u([1.0, 7.0, float("inf"), -1.0, float("nan")])[:, 0]
    assert x[:4].tolist() == [1.0, 7.0, float("inf"), -1.0] and torch.isnan(x[4])


def test_numbers_of_32_bits_are_as_they_are():
    u = torch.rand((9, 3), generator=torch.Generator().manual_seed(1))
    assert torch.equal(_u(u, rows=3), u) and torch.equal(_u(u.t().contiguous().t(), rows=3), u)
