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


@pytest.mark.parametrize("kv_type", [F16, Q8_0])
def test_a_prompt_longer_than_the_cache_under_a_window(exact, kv_type):  # noqa: F811
    """Six pages of 32 positions: a prompt of 200 tokens beside a decoding sequence, as with room for all of it; one that
    fails on the way leaves both as they were."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model("mixtral_like_hd128", n_batch=16)
    rng = np.random.default_rng(8)
    toks, more = rng.integers(0, 600, 200).tolist(), rng.integers(0, 600, 45).tolist()
    small = PagedDecoder(exact, hp, T, 7, 32, kv_type, 40, 3)
    large = PagedDecoder(exact, hp, T, 30, 32, kv_type, 40, 3, layer_base=2000)
    try:
        for rows in ({1: toks[:20]}, {0: toks, 1: [5]}, {1: [6], 0: [7]}):
            a, b = (host(d.forward(rows)) for d in (small, large))
            _near(a, b)
        assert small.account.usage()[0] == large.account.usage()[0] <= 6
        count, rows_of = [0], small._rows

        def third(x, batch):
            count[0] += 1
            if count[0] == 3:
                raise RuntimeError("no")
            return rows_of(x, batch)

        small._rows = third
        with pytest.raises(RuntimeError):
            small.forward({0: more, 4: [9]})
        small._rows = rows_of
        assert [small.length(s) for s in (0, 1, 4)] == [201, 22, 0]
        with pytest.raises(KmoeError):  # four sequences' windows do not fit
            small.forward({s: more for s in (0, 1, 2, 3)})
        assert [small.length(s) for s in range(4)] == [201, 22, 0, 0]
        a, b = (host(d.forward({0: [1], 1: [2]})) for d in (small, large))
        _near(a, b)
    finally:
        small.close()
        large.close()


@pytest.mark.parametrize("use_graph", [True, False])
def test_a_generation_longer_than_the_cache_under_a_window(exact, use_graph):  # noqa: F811
    """Greedy steps past the pages: the tokens of single steps with room for all of them."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model()
    toks = {s: np.random.default_rng(s).integers(0, 1000, 5 + 20 * s).tolist() for s in (1, 2)}
    # of each at once: the pages up to its end before the call (1 and 2), two of a window and the next block's; all
    # positions take 6 and 7
    small = PagedDecoder(exact, hp, T, 10, 32, F16, 33, 2)
    large = PagedDecoder(exact, hp, T, 30, 32, F16, 33, 2)
    try:
        for d in (small, large):
            d.forward(toks)
        f, want = {1: 11, 2: 12}, []
        for _ in range(150):
            f = dict(zip(f, np.argmax(host(large.forward({s: [t] for s, t in f.items()})), 1).tolist()))
            want.append(list(f.values()))
        got = host(small.decode_greedy({1: 11, 2: 12}, 150, use_graph=use_graph)).tolist()
        assert got == want
        assert [small.length(s) for s in (1, 2)] == [175, 195] and small.account.usage() == (large.account.usage()[0], 10)
    finally:
        small.close()
        large.close()
