"""PagedDecoder: the paged cache's operators together, as a server uses them
(kestrel_amd.decoder): prompts and single tokens of several sequences in one
call, forks, windows with trimming, compaction, a full cache, greedy steps as
a captured graph; against the oracle's Transformer::forward
(transformer.rs:278-302) per sequence."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0, KmoeError
from tests.helpers import decoder_model, rel_l2
from tests.test_gpu_decoder import MODELS, ctx, host  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def exact(ctx):  # noqa: F811
    ctx.set_regime(2)
    yield ctx
    ctx.set_regime(0)


def _model(name="llama_dense", seed=3, **more):
    return decoder_model(seed=seed, **{**MODELS[name], **more})


def _near(a, b):
    """The bounds of the single-sequence Decoder's test in the exact regime."""
    scale = max(1.0, float(np.abs(b).max()))
    assert rel_l2(a, b) < 1e-3 and float(np.abs(a - b).max()) <= 2e-3 * scale, (rel_l2(a, b), scale)


@pytest.mark.parametrize("name", list(MODELS))
def test_mixed_batches_match_the_oracle(exact, orc, name):
    """Prompts of 1, 9 and 40 tokens together, then single tokens beside a new prompt, one sequence sitting out."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model(name)
    V = T["token_embd.weight"][1][1]
    rng = np.random.default_rng(1)
    draw = lambda n: rng.integers(0, V, n).tolist()  # noqa: E731
    calls = [{7: draw(9), 2: draw(1), 5: draw(40)}, {5: draw(1), 7: draw(1)}, {2: draw(1), 9: draw(33), 5: draw(1)},
             {9: draw(1), 7: draw(1), 2: draw(1), 5: draw(1)}]
    dec = PagedDecoder(exact, hp, T, n_pages=8, page=32)
    refs = {s: orc.Transformer(hp, T, regime=2) for s in (2, 5, 7, 9)}
    try:
        for rows in calls:
            got = host(dec.forward(rows))
            assert got.shape == (len(rows), V)
            for a, (s, ts) in zip(got, rows.items()):
                _near(a, refs[s].forward(ts))
        assert [dec.length(s) for s in (2, 5, 7, 9, 1)] == [3, 43, 11, 34, 0]
    finally:
        dec.close()


@pytest.mark.parametrize("kv_type", [F16, Q8_0])
def test_a_fork_writes_on_pages_of_its_own(exact, orc, kv_type):
    """Two forks inside a page go on with other tokens than their origin; each as if it had been fed alone."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model()
    rng = np.random.default_rng(2)
    p = rng.integers(0, 1000, 45).tolist()
    dec = PagedDecoder(exact, hp, T, n_pages=12, page=32, kv_type=kv_type)
    alone = PagedDecoder(exact, hp, T, n_pages=16, page=32, kv_type=kv_type)
    try:
        dec.forward({0: p})
        dec.fork(0, 1)
        dec.fork(0, 2, 37)
        assert dec.account.usage()[0] == 2
        rows = {2: [11], 0: [12, 13], 1: [14]}
        got = [host(dec.forward(rows)), host(dec.forward({0: [15], 1: [16], 2: [17]}))]
        fed = {0: p + [12, 13], 1: p + [14], 2: p[:37] + [11]}
        for i, s in enumerate(rows):
            _near(got[0][i], host(alone.forward({10 + s: fed[s]}))[0])
        for s in range(3):
            _near(got[1][s], host(alone.forward({10 + s: [15 + s]}))[0])
        if kv_type == F16:
            _near(got[1][1], orc.Transformer(hp, T, regime=2).forward(fed[1] + [16]))
        dec.drop(0)
        dec.drop(1)
        dec.drop(2)
        assert dec.account.usage()[0] == 0
    finally:
        dec.close()
        alone.close()


@pytest.mark.parametrize("kv_type", [F16, Q8_0])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (40, 0), (33, 5), (1000, 3)])
def test_chunks_windows_and_trimming(exact, kv_type, window, n_sink):
    """A prompt in one call, and the same by parts with pages trimmed on the way: the same logits, and no more pages
    held than the window needs."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model("mixtral_like_hd128", n_batch=64)
    toks = np.random.default_rng(3).integers(0, 600, 200).tolist()
    one = PagedDecoder(exact, hp, T, 8, 32, kv_type, window, n_sink)
    hp2 = dict(hp, n_batch=4)
    two = PagedDecoder(exact, hp2, T, 8, 32, kv_type, window, n_sink, layer_base=2000)
    try:
        a = host(one.forward({0: toks}))[0]
        i = 0
        for n in (1, 50, 3, 1, 1, 70, 7, 1, 66):
            b = host(two.forward({0: toks[i:i + n]}))[0]
            i += n
            if 0 < window < 200:
                assert two.account.usage()[0] <= -(-window // 32) + 1 + (n_sink > 0)
        assert i == 200 and two.account.usage()[0] == one.account.usage()[0]
        _near(b, a)
    finally:
        one.close()
        two.close()


def test_compaction_and_truncation_change_no_bits(exact):
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model()
    rng = np.random.default_rng(4)
    toks = {s: rng.integers(0, 1000, 30 + 20 * s).tolist() for s in range(4)}
    out = []
    for compact in (False, True):
        dec = PagedDecoder(exact, hp, T, 16, 32)
        try:
            dec.forward(toks)
            dec.drop(0)
            dec.drop(2)
            if compact:
                assert dec.compact() > 0
                assert dec.account.table([1, 3], 4)[0].max() < dec.account.usage()[0]
            dec.forward({1: [5, 6, 7], 3: [8]})
            dec.truncate(1, 51)
            out.append(host(dec.forward({3: [1], 1: [2]})))
        finally:
            dec.close()
    assert np.array_equal(out[0].view(np.uint32), out[1].view(np.uint32))


def test_a_full_cache_refuses_and_changes_nothing(exact, orc):
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model()
    rng = np.random.default_rng(5)
    p = rng.integers(0, 1000, 40).tolist()
    dec = PagedDecoder(exact, hp, T, 4, 32)
    ref = orc.Transformer(hp, T, regime=2)
    try:
        dec.forward({0: p})
        dec.fork(0, 1)
        with pytest.raises(KmoeError):  # 0 gets a page of its own first, 2 finds none
            dec.forward({0: [1], 2: p + p})
        assert [dec.length(s) for s in (0, 1, 2)] == [40, 40, 0]
        for bad in ({0: []}, {0: [1000]}, {0: [-1]}, {0: [1] * 217}, {}):
            with pytest.raises(ValueError):
                dec.forward(bad)
        with pytest.raises(ValueError):
            dec.decode_greedy({0: 1}, 217)
        with pytest.raises(ValueError):
            dec.decode_greedy({0: 1}, 0)
        with pytest.raises(KmoeError):
            dec.decode_greedy({0: 1, 1: 1}, 60)
        assert [dec.length(s) for s in (0, 1)] == [40, 40]
        ref.forward(p)
        want = ref.forward([9])
        got = host(dec.forward({0: [9], 1: [9]}))
        _near(got[0], want)
        _near(got[1], want)
    finally:
        dec.close()


@pytest.mark.parametrize("name", ["llama_dense", "qwen3moe"])
@pytest.mark.parametrize("regime", [2, 0])
@pytest.mark.parametrize("kv_type", [F16, Q8_0])
def test_greedy_graph_gives_the_tokens_of_single_steps(ctx, name, regime, kv_type):  # noqa: F811
    """Several sequences decoded together: captured and replayed, eager, and step by step through forward with the
    argmax on the host; twice from the same graph, with eager work between and with other sequences."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model(name)
    V = T["token_embd.weight"][1][1]
    rng = np.random.default_rng(6)
    toks = {s: rng.integers(0, V, n).tolist() for s, n in enumerate((3, 50, 17, 31, 64))}
    outs = []
    ctx.set_regime(regime)
    try:
        for how in ("graph", "eager", "steps"):
            dec = PagedDecoder(ctx, hp, T, 32, 32, kv_type, window=48, n_sink=2)
            try:
                first = np.argmax(host(dec.forward(toks)), 1)
                got = []
                for seqs, n in (((0, 1, 2, 3), 7), ((4, 2, 0, 1), 5)):
                    f = {s: int(first[s]) for s in seqs}
                    if how == "steps":
                        for _ in range(n):
                            f = dict(zip(f, np.argmax(host(dec.forward({s: [t] for s, t in f.items()})), 1).tolist()))
                            got.append(list(f.values()))
                    else:
                        got += host(dec.decode_greedy(f, n, use_graph=how == "graph")).tolist()
                    dec.forward({3: [1, 2, 3]})
                outs.append((got, [dec.length(s) for s in range(5)], dec.account.usage()[0]))
            finally:
                dec.close()
    finally:
        ctx.set_regime(0)
    assert outs[0] == outs[1] == outs[2]


def test_constructor_refusals(exact):
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model()
    for more in (dict(kv_type=2), dict(window=-1), dict(n_sink=3), dict(window=5, n_sink=-1), dict(page=48)):
        with pytest.raises(ValueError):
            PagedDecoder(exact, hp, T, 4, **more)
    with pytest.raises(ValueError):
        PagedDecoder(exact, dict(hp, head_dim=32), T, 4)
    with pytest.raises(KmoeError):
        PagedDecoder(exact, hp, T, 0)
