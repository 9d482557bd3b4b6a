"""PagedDecoder's calls as wholes: those that fail leave the sequences as they were, and a window's pages serve prompts
and generations longer than the cache."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0, KmoeError  # noqa: F401
from tests.test_gpu_decoder import ctx, host  # noqa: F401  (ctx: a fixture)
from tests.test_gpu_paged_decoder import _model, _near, exact  # noqa: F401  (exact: a fixture)

pytestmark = pytest.mark.gpu


def test_a_call_that_fails_at_its_end(exact, monkeypatch):  # noqa: F811
    """No memory for the logits of several parts: the sequences are as before the call, and go on."""
    import torch

    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model(n_batch=8)
    dec, ref = PagedDecoder(exact, hp, T, 16, 32), PagedDecoder(exact, hp, T, 16, 32, layer_base=2000)

    def none(*a, **k):
        raise torch.cuda.OutOfMemoryError("no memory")

    try:
        for d in (dec, ref):
            d.forward({0: [1, 2, 3], 1: [4]})
        with monkeypatch.context() as m:
            m.setattr(torch, "cat", none)
            with pytest.raises(torch.cuda.OutOfMemoryError):
                dec.forward({0: [5] * 7, 1: [6] * 5, 2: [7]})
        assert [dec.length(s) for s in range(3)] == [3, 1, 0] and dec.account.usage() == ref.account.usage()
        a, b = (host(d.forward({1: [8], 0: [9]})) for d in (dec, ref))
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    finally:
        dec.close()
        ref.close()
