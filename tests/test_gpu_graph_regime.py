"""A decoder's captured greedy step follows the context's regime."""
import numpy as np
import pytest

from tests.helpers import decoder_model
from tests.test_gpu_decoder import MODELS, ctx, host  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["llama_dense", "qwen3moe"])
@pytest.mark.parametrize("paged", [False, True])
def test_a_change_of_regime_captures_anew(ctx, name, paged):  # noqa: F811
    """Greedy steps in the exact regime, then in the AVX2 regime and back, on one decoder: the logits of the replayed
    steps are those of eager ones, bit for bit."""
    from kestrel_amd.decoder import Decoder, PagedDecoder

    hp, T = decoder_model(seed=5, **MODELS[name])
    toks = np.random.default_rng(1).integers(0, T["token_embd.weight"][1][1], 9).tolist()
    runs = []
    try:
        for use_graph in (True, False):
            dec = PagedDecoder(ctx, hp, T, n_pages=8, page=32) if paged else Decoder(ctx, hp, T)
            try:
                got = []
                ctx.set_regime(2)
                dec.forward({0: toks} if paged else toks)
                for regime in (2, 0, 0, 2):
                    ctx.set_regime(regime)
                    dec.decode_greedy({0: 7} if paged else 7, 2, use_graph=use_graph)
                    got.append(host(dec._graph_bufs["logits"]).reshape(-1).view(np.uint32).copy())
                runs.append(got)
            finally:
                dec.close()
    finally:
        ctx.set_regime(0)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))
