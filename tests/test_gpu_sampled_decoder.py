"""Sampled decoding, shared prefixes and selected pages in the decoders, as a server
uses them together: a prompt fed once, forks that go on by drawn tokens, long contexts
of which a few pages are read (kestrel_amd.decoder)."""
import numpy as np
import pytest

from kestrel_amd.kmoe import F16, Q8_0, KmoeError
from tests.test_gpu_decoder import ctx, host  # noqa: F401  (ctx: a fixture)
from tests.test_gpu_paged_decoder import _model, _near, exact  # noqa: F401  (exact: a fixture)

pytestmark = pytest.mark.gpu


def _sample(ctx, logits, u, temperature, top_k, top_p, min_p):  # noqa: F811
    """Context.sample with settings of the host."""
    import torch

    S = len(logits)
    d = lambda v, t: torch.from_numpy(np.broadcast_to(np.asarray(v, t), S).copy()).cuda()  # noqa: E731
    return host(ctx.sample(logits, d(u, np.float32), d(temperature, np.float32), d(top_k, np.int32), d(top_p, np.float32), d(min_p, np.float32)))


@pytest.mark.parametrize("name", ["llama_dense", "qwen3moe"])
@pytest.mark.parametrize("regime", [2, 0])
def test_one_sequence(ctx, name, regime):  # noqa: F811
    """Captured, eager, and step by step through forward; twice from one graph with other settings, a greedy graph beside it."""
    from kestrel_amd.decoder import Decoder

    hp, T = _model(name)
    V = T["token_embd.weight"][1][1]
    rng = np.random.default_rng(1)
    prompt, u = rng.integers(0, V, 9).tolist(), rng.random((2, 6)).astype(np.float32)
    hows = [dict(temperature=0.9, top_k=50, top_p=0.95, min_p=0.0), dict(temperature=1.7, top_k=0, top_p=1.0, min_p=0.01)]
    outs = []
    ctx.set_regime(regime)
    try:
        for how in ("graph", "eager", "steps"):
            dec = Decoder(ctx, hp, T)
            try:
                dec.forward(prompt)
                got, t = [], 5
                for x, h in zip(u, hows):
                    if how == "steps":
                        for i in range(6):
                            t = int(_sample(ctx, dec.forward([t]).view(1, -1), x[i], **h)[0])
                            got.append(t)
                        for i in range(2):
                            t = int(np.argmax(host(dec.forward([t]))))
                            got.append(t)
                    else:
                        got += host(dec.decode_sample(t, 6, x, **h, use_graph=how == "graph")).tolist()
                        got += host(dec.decode_greedy(got[-1], 2, use_graph=how == "graph")).tolist()
                        t = got[-1]
                outs.append((got, dec.cached))
            finally:
                dec.close()
    finally:
        ctx.set_regime(0)
    assert outs[0] == outs[1] == outs[2]


@pytest.mark.parametrize("form", ["plain", "shared", "selected", "window"])
@pytest.mark.parametrize("kv_type", [F16, Q8_0])
def test_many_sequences(ctx, form, kv_type):  # noqa: F811
    """A prompt, its forks and a sequence of its own, decoded together by settings of each one's own: captured, eager and
    step by step; then other sequences, then greedily."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model("llama_dense")
    more = dict(plain={}, shared=dict(share_prefixes=True), selected=dict(select=3, select_first=1), window=dict(window=48, n_sink=2))[form]
    rng = np.random.default_rng(2)
    prompt, other = rng.integers(0, 1000, 150).tolist(), rng.integers(0, 1000, 20).tolist()
    runs = [({0: 3, 9: 4, 2: 5, 1: 6, 3: 7}, 5), ({2: 1, 0: 2, 9: 3}, 4)]
    outs = []
    for how in ("graph", "eager", "steps"):
        dec = PagedDecoder(ctx, hp, T, 64, 32, kv_type, **more)
        rng = np.random.default_rng(3)
        try:
            dec.SHARE_LEAST = 64
            dec.forward({0: prompt})
            dec.forward({9: other})
            for s, n in ((1, 150), (2, 131), (3, 150)):
                dec.fork(0, s, 150 if form == "window" else n)  # (under a window an earlier position is given up)
            got = []
            for first, n in runs:
                S = len(first)
                h = dict(temperature=rng.choice([0.0, 0.7, 1.5], S), top_k=rng.choice([0, 1, 30], S), top_p=rng.choice([1.0, 0.9], S), min_p=0.001)
                u = rng.random((n, S))
                if how == "steps":
                    f = dict(first)
                    for i in range(n):
                        f = dict(zip(f, _sample(ctx, dec.forward({s: [t] for s, t in f.items()}), u[i], **h).tolist()))
                        got.append(list(f.values()))
                    for _ in range(2):
                        f = dict(zip(f, np.argmax(host(dec.forward({s: [t] for s, t in f.items()})), 1).tolist()))
                        got.append(list(f.values()))
                else:
                    o = host(dec.decode_sample(first, n, u, **h, use_graph=how == "graph"))
                    assert o.shape == (n, S)
                    got += o.tolist()
                    got += host(dec.decode_greedy(dict(zip(first, o[-1].tolist())), 2, use_graph=how == "graph")).tolist()
            outs.append((got, [dec.length(s) for s in (0, 1, 2, 3, 9)], dec.account.usage()[0]))
        finally:
            dec.close()
    assert outs[0] == outs[1] == outs[2]


@pytest.mark.parametrize("kv_type", [F16, Q8_0])
def test_shared_prefixes_change_no_logits(exact, orc, kv_type):  # noqa: F811
    """Forks of two prompts, mixed chunks and single tokens, with and without sharing; the order of the answers is the
    caller's; against the oracle per sequence with F16."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model("mixtral_like_hd128")
    V = T["token_embd.weight"][1][1]
    rng = np.random.default_rng(4)
    draw = lambda n: rng.integers(0, V, n).tolist()  # noqa: E731
    p = {0: draw(100), 50: draw(70)}
    calls = [{3: draw(1), 50: draw(2), 1: draw(1), 0: draw(1), 51: draw(30), 2: draw(4), 7: draw(5)},
             {0: draw(1), 51: draw(1), 7: draw(1), 2: draw(1), 3: draw(1), 50: draw(1), 1: draw(1)},
             {2: draw(40), 3: draw(1)}]
    outs, seen = [], {}
    for share in (True, False):
        dec = PagedDecoder(exact, hp, T, 64, 32, kv_type, share_prefixes=share)
        try:
            dec.SHARE_LEAST = 1
            dec.forward(p)
            for src, dst, n in ((0, 1, 100), (0, 2, 97), (0, 3, 64), (50, 51, 69)):
                dec.fork(src, dst, n)
                seen[dst] = p[src][:n]
            if share:
                assert len(dec._groups([0, 1, 2, 3, 50, 51], 6)[2]) == 2
            outs.append([host(dec.forward(c)) for c in calls])
        finally:
            dec.close()
    for a, b in zip(*outs):
        _near(a, b)
    if kv_type == F16:
        for s, base in ((1, p[0]), (3, seen[3]), (51, seen[51])):
            ref = orc.Transformer(hp, T, regime=2)
            ref.forward(base)
            for c, got in zip(calls, outs[0]):
                if s in c:
                    _near(got[list(c).index(s)], ref.forward(c[s]))


@pytest.mark.parametrize("kv_type", [F16, Q8_0])
def test_bounds_stay_those_of_the_pages(exact, kv_type):  # noqa: F811
    """Through prompts, forks, truncations, decoding and compaction: whole pages' bounds are what they are formed anew as."""
    import torch
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model("llama_dense")
    rng = np.random.default_rng(5)
    draw = lambda n: rng.integers(0, 1000, n).tolist()  # noqa: E731
    dec = PagedDecoder(exact, hp, T, 40, 32, kv_type, select=3)
    try:
        dec.forward({0: draw(130), 1: draw(40), 5: draw(70)})
        dec.fork(0, 2, 110)
        dec.forward({2: draw(1), 0: draw(1)})
        dec.truncate(0, 50)
        dec.forward({0: draw(60), 1: draw(1)})
        dec.decode_greedy({0: 1, 1: 2, 2: 3}, 40)
        dec.drop(5)
        assert dec.compact() > 0
        dec.decode_sample({2: 1, 1: 2}, 20, rng.random((20, 2)), top_k=20)
        seqs = [0, 1, 2]
        t, n = dec.account.table(seqs, dec.cols)
        start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        d = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()  # noqa: E731
        b = exact.paged_batch(d(t), d(n), d(start), int(start[-1]))
        for l in range(dec.n_layer):
            want = exact.paged_bounds(dec.kv, dec.pages[l], b, torch.zeros_like(dec.bounds[l]))
            for i in range(3):
                ids = t[i, :n[i] // 32].tolist()
                assert ids and torch.equal(dec.bounds[l][ids], want[ids])
    finally:
        dec.close()


def test_selection_of_all_pages_and_of_few(exact):  # noqa: F811
    """With as many pages as there are the logits are the plain decoder's; with few, compaction changes no bits, and prompts
    are read whole."""
    from kestrel_amd.decoder import PagedDecoder

    hp, T = _model("llama_dense")
    rng = np.random.default_rng(6)
    prompt = rng.integers(0, 1000, 200).tolist()
    steps = [{0: [int(t)], 1: [7]} for t in rng.integers(0, 1000, 5)]
    outs = []
    for more, compact in ((dict(), False), (dict(select=7), False), (dict(select=2, select_first=0), False), (dict(select=2, select_first=0), True)):
        dec = PagedDecoder(exact, hp, T, 30, 32, **more)
        try:
            dec.forward({3: prompt[:70]})
            got = [host(dec.forward({0: prompt, 1: prompt[:90]}))]
            dec.drop(3)
            if compact:
                assert dec.compact() > 0
            got += [host(dec.forward(c)) for c in steps]
            outs.append(got)
        finally:
            dec.close()
    for a, b in zip(outs[0], outs[1]):
        _near(a, b)
    assert np.array_equal(outs[0][0], outs[2][0])
    assert any(np.abs(a - b).max() > 1e-3 for a, b in zip(outs[0][1:], outs[2][1:]))  # (it does leave pages out)
    assert all(np.array_equal(a, b) for a, b in zip(outs[2], outs[3]))


def test_refusals(exact):  # noqa: F811
    from kestrel_amd.decoder import Decoder, PagedDecoder

    hp, T = _model()
    for more in (dict(select=-1), dict(select=2, select_first=2), dict(select=2, select_first=-1), dict(select=4, window=9),
                 dict(share_prefixes=True, window=9), dict(share_prefixes=True, select=4)):
        with pytest.raises(ValueError):
            PagedDecoder(exact, hp, T, 4, **more)
    dec, one = PagedDecoder(exact, hp, T, 4, 32), Decoder(exact, hp, T, layer_base=2000)
    try:
        dec.forward({0: [1, 2, 3], 1: [4]})
        one.forward([1, 2])
        u = np.full((3, 2), 0.5)
        for bad in (dict(u=u[:2]), dict(u=u[:, :1]), dict(u=0.5), dict(u=u[:, 0]), dict(u=u, temperature=[1.0]), dict(u=u, top_k=[1, 2, 3]),
                    dict(u=u, top_p=np.ones((2, 1))), dict(u=u, min_p=[[0, 0]])):
            with pytest.raises(ValueError):
                dec.decode_sample({0: 5, 1: 6}, 3, **bad)
        with pytest.raises(ValueError):
            dec.decode_sample({0: 5, 1: 1000}, 3, u)
        with pytest.raises(KmoeError):
            dec.decode_sample({0: 5, 1: 6}, 90, np.full((90, 2), 0.5))
        assert [dec.length(s) for s in (0, 1)] == [3, 1]
        for bad in (dict(u=u), dict(u=[0.5] * 2), dict(u=[0.5] * 3, top_k=[1, 2])):
            with pytest.raises(ValueError):
                one.decode_sample(5, 3, **bad)
        with pytest.raises(ValueError):
            one.decode_sample(5, 10 ** 6, [0.5])
        assert one.cached == 2
        assert one.decode_sample(5, 3, [0.5] * 3, top_k=[4]).shape == (3,) and one.cached == 5
        assert dec.decode_sample({0: 5, 1: 6}, 3, u.tolist(), temperature=[0.5, 2], top_k=10 ** 12).shape == (3, 2)
    finally:
        dec.close()
        one.close()
