"""Timed cases of what a server that draws many continuations over a paged
key-value cache needs besides its store and its attention: sampling of the next
tokens, attention of sequences that share a long prefix, the bounds of a page's
keys, and attention over the pages that those bounds select.

listed() names the cases, draw() gives more of the same ranges, prepare() makes
what such a program holds before the call, run() is one pass, work() the bytes
and operations it cannot do without, exact() the same outputs in 64 bits.

With `own` false run() takes elementary torch operations, with `own` true the
calls of kestrel_amd.kmoe.Context.

sample    w_i = exp((l_i - max l) / T), T > 0. In the order of descending l
          (equal ones by index) the first top_k tokens are kept, of those the
          shortest beginning that holds top_p of their weight, of those the ones
          with w_i >= min_p. The token drawn is the first kept one, by index, at
          which the running sum of w passes u times the sum of all kept. T <= 0:
          the first largest.
shared    causal attention of rows over their sequences' pages; the sequences of
          a group have their first pages in common.
bounds    per page, kv head and dim, the least and the largest key among the
          sequence's positions on the page (f16).
selected  causal attention, per row and kv head over a few pages: the row's own
          one, the first `first` ones, and those with the largest
          sum_heads sum_dims max(q lo, q hi) (64 bits; equal ones: the lower
          position), `select` pages in all.

A page holds `page` positions of every kv head of one layer. Its bytes, per kv
head (offsets _k_at .. _vs_at below):
  f16   K in tiles of 16 positions x 32 dims, then V in tiles of 16 dims x 32
        positions, both two bytes an element
  q8_0  one byte an element in the same tiles, two of them side by side, and
        one f16 scale per position and 32 dims, after K's bytes and after V's
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # one chat: the usual settings, one row of logits
        dict(name="sample-1", kind="sample", rows=1, vocab=32000, how="one", temp=0.8, k=40, p=0.95, m=0.0, peak=9.0),
        # a server's step: every sequence with settings of its own, greedy ones among them
        dict(name="sample-64-mixed", kind="sample", rows=64, vocab=102400, how="mixed", temp=0.0, k=0, p=0.0, m=0.0, peak=8.0),
        # many continuations drawn from the whole distribution
        dict(name="sample-256-plain", kind="sample", rows=256, vocab=151936, how="one", temp=1.0, k=0, p=1.0, m=0.0, peak=6.0),
        # a hot nucleus over a flat distribution: thousands of tokens are kept
        dict(name="sample-16-flat", kind="sample", rows=16, vocab=151936, how="one", temp=1.3, k=0, p=0.9, m=0.0, peak=0.0),
        # eight continuations of a short prompt
        dict(name="shared-8-at-1000", kind="shared", t="f16", heads=16, kv=4, hd=128, page=64, groups=1, members=8, alone=0,
             lo=1000, hi=1000, tail=60, rows=1),
        # 64 continuations of a document
        dict(name="shared-64-at-6000", kind="shared", t="f16", heads=32, kv=8, hd=128, page=64, groups=1, members=64, alone=0,
             lo=6000, hi=6000, tail=300, rows=1),
        # several system prompts, sequences of their own beside them, a few drafted tokens per step, 8-bit cache
        dict(name="shared-groups-q8", kind="shared", t="q8_0", heads=16, kv=8, hd=64, page=32, groups=5, members=17, alone=11,
             lo=500, hi=4000, tail=500, rows=3),
        # the pages that a decode step's new rows lie on
        dict(name="bounds-64", kind="bounds", t="f16", heads=32, kv=8, hd=128, page=64, seqs=64, lo=100, hi=8192, prompts=0, rows=1),
        # a prompt's pages, 8-bit cache
        dict(name="bounds-1777-q8", kind="bounds", t="q8_0", heads=16, kv=4, hd=128, page=32, seqs=1, lo=1777, hi=1777,
             prompts=1, rows=1777),
        # one token over a very long context, 64 pages of 2047
        dict(name="selected-1-at-131000", kind="selected", t="f16", heads=32, kv=8, hd=128, page=64, seqs=1, lo=131000,
             hi=131000, prompts=0, rows=1, select=64, first=1),
        # a decode step of chats of very different lengths, some shorter than the selection
        dict(name="selected-48-q8", kind="selected", t="q8_0", heads=32, kv=8, hd=128, page=64, seqs=48, lo=300, hi=9000,
             prompts=0, rows=1, select=32, first=1),
        # a chunk of a long prompt
        dict(name="selected-chunk-300", kind="selected", t="f16", heads=16, kv=4, hd=128, page=64, seqs=1, lo=16000, hi=16000,
             prompts=1, rows=300, select=24, first=2),
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _padded(c):
    """Elements of K over all sequences, each at the longest one's length."""
    lens = _lens(c)
    return len(lens) * max(lens) * c["kv"] * c["hd"]


def _too_much(c):
    """Past the largest listed case of its kind, or past a few GB where the plain form pads to the longest sequence."""
    if _cost(c) > max(_cost(x) for x in listed() if x["kind"] == c["kind"]):
        return True
    if c["kind"] in ("sample", "bounds"):
        return False
    return _padded(c) > 430_000_000 or _padded(c) * max(_rows(c)) * c["heads"] // (c["kv"] * c["hd"]) > 200_000_000


def draw(rng):
    kind = rng.choice(["sample", "sample", "sample", "shared", "shared", "shared", "selected", "selected", "selected", "bounds"])
    if kind == "sample":
        c = dict(kind="sample", rows=_between(rng, 1, 300), vocab=_between(rng, 500, 200000), how=rng.choice(["one", "one", "mixed"]),
                 temp=round(rng.uniform(0.3, 1.6), 3), k=rng.choice([0, 0, 1, _between(rng, 2, 1000)]),
                 p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]), m=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]),
                 peak=rng.choice([0.0, round(rng.uniform(3.0, 12.0), 2)]))
        while _too_much(c):
            c["rows"] = max(1, c["rows"] // 2)
        return c
    t, page = rng.choice(["f16", "f16", "q8_0"]), rng.choice([32, 64, 128, 256])
    heads, kv, hd = rng.choice([(16, 4, 128), (32, 8, 128), (16, 16, 128), (16, 8, 64), (12, 4, 64), (14, 2, 64), (32, 2, 128)])
    c = dict(kind=kind, t=t, heads=heads, kv=kv, hd=hd, page=page)
    if kind == "shared":
        c |= dict(groups=_between(rng, 1, 12), members=_between(rng, 2, 80), alone=rng.choice([0, 0, 1, _between(rng, 1, 30)]),
                  lo=1, hi=_between(rng, 100, 20000), tail=_between(rng, 1, 2000), rows=rng.choice([1, 1, 1, _between(rng, 2, 40)]))
    else:
        form = rng.choice(["decode", "decode", "prompt", "mixed"])
        c |= dict(seqs=1 if rng.random() < 0.2 else _between(rng, 1, 128 if form == "decode" else 8), lo=1,
                  hi=_between(rng, 40, 131000 if kind == "selected" else 16384), prompts=0, rows=1)
        if form != "decode":
            c["prompts"] = c["seqs"] if form == "prompt" else rng.randint(1, c["seqs"])
            c["rows"] = _between(rng, 2, 500 if kind == "selected" else 2000)
        if kind == "selected":
            c["select"] = _between(rng, 2, 128)
            c["first"] = rng.randint(0, min(4, c["select"] - 1))
    c["lo"] = _between(rng, 1, c["hi"])
    while _too_much(c):
        many = "members" if kind == "shared" else "seqs"
        if kind == "shared" and c["groups"] > 1 and rng.random() < 0.4:
            c["groups"] //= 2
        elif c["rows"] > 1 and rng.random() < 0.4:
            c["rows"] //= 2
        elif c[many] > (2 if kind == "shared" else 1) and rng.random() < 0.6:
            c[many] = max(2 if kind == "shared" else 1, c[many] // 2)
            if kind != "shared":
                c["prompts"] = min(c["prompts"], c["seqs"])
        else:
            c["hi"] = max(2, c["hi"] // 2)
            c["lo"] = min(c["lo"], c["hi"])
            if kind == "shared":
                c["tail"] = max(1, c["tail"] // 2)
    return c


def _spread(lo, hi, n):
    """n whole numbers evenly over the logarithm of lo..hi, the smallest first."""
    if n == 1:
        return [hi]
    a, b = math.log(lo), math.log(hi)
    return [min(hi, max(lo, int(round(math.exp(a + (b - a) * i / (n - 1)))))) for i in range(n)]


def _shared_pages(c):
    """Pages that each group has in common (whole ones of its prefix)."""
    return [n // c["page"] for n in _spread(c["lo"], c["hi"], c["groups"])]


def _lens(c):
    """The sequences' lengths."""
    if c["kind"] != "shared":
        return _spread(c["lo"], c["hi"], c["seqs"])
    # behind the prefix's whole pages: what is left of it, and 1 .. tail positions of its own (rows at least)
    own_ = [c["rows"] + (i * 37) % c["tail"] for i in range(c["members"])]
    lens = [n + x for n in _spread(c["lo"], c["hi"], c["groups"]) for x in own_]
    return lens + [c["rows"] + x for x in _spread(1, c["hi"], max(1, c["alone"]))][:c["alone"]]


def _rows(c):
    """New rows of each sequence: chunks of `rows` for the longest ones, one for the others (shared: `rows` each)."""
    n = _lens(c)
    if c["kind"] == "shared":
        return [c["rows"]] * len(n)
    return [min(c["rows"], x) if i >= c["seqs"] - c["prompts"] else 1 for i, x in enumerate(n)]


# ------------------------------------------------------------- page layout

def _block_bytes(c):
    """Bytes of one kv head in a page."""
    return 2 * c["page"] * c["hd"] * 2 if c["t"] == "f16" else 2 * (c["page"] * c["hd"] + c["page"] * (c["hd"] // 32) * 2)


def _page_bytes(c):
    return c["kv"] * _block_bytes(c)


def _k_at(c, p, d):
    """Element of K (position p of the page, dim d) within the kv head's bytes, counted in elements."""
    hd = c["hd"]
    if c["t"] == "f16":
        return ((p // 16) * (hd // 32) + d // 32) * 512 + (d % 32) // 8 * 128 + p % 16 * 8 + d % 8
    return p // 16 * (16 * hd) + d // 64 * 1024 + (d % 32) // 8 * 256 + p % 16 * 16 + d // 32 % 2 * 8 + d % 8


def _v_at(c, p, d):
    hd, r = c["hd"], p % 32
    g, j = r % 16 // 4, r % 4 + 4 * (r // 16)
    if c["t"] == "f16":
        return c["page"] * hd + p // 32 * (32 * hd) + d // 16 * 512 + g * 128 + d % 16 * 8 + j
    return c["page"] * hd + c["page"] * (hd // 32) * 2 + p // 32 * (32 * hd) + d // 32 * 1024 + g * 256 + d % 16 * 16 + d // 16 % 2 * 8 + j


def _ks_at(c, p, u):
    """Byte of the f16 scale of position p, dims 32 u .. 32 u + 31, in q8_0 pages."""
    n = c["hd"] // 32
    return c["page"] * c["hd"] + 2 * (p // 16 * (16 * n) + p % 16 // 4 * (4 * n) + u * 4 + p % 4)


def _vs_at(c, p, u):
    n, r = c["hd"] // 32, p % 32
    return _block_bytes(c) - 2 * c["page"] * n + 2 * (p // 32 * (32 * n) + r % 16 // 4 * (8 * n) + u * 8 + r % 4 + 4 * (r // 16))


def _blocks(s, ids):
    """K and V [..., kv, page, hd] in 32 bits of the pages `ids` [...]."""
    c = s["case"]
    kv, hd, pg = c["kv"], c["hd"], c["page"]
    sh = tuple(ids.shape) + (kv,)
    x = s["pages"].view(s["n_pages"], kv, _block_bytes(c))[ids.reshape(-1)]
    n, N = hd // 32, x.shape[0] * kv
    x = x.view(N, -1)
    if c["t"] == "f16":
        x = x.view(torch.float16)
        k = x[:, :pg * hd].view(N, pg // 16, n, 4, 16, 8).permute(0, 1, 4, 2, 3, 5)
        v = x[:, pg * hd:].view(N, pg // 32, hd // 16, 4, 16, 2, 4).permute(0, 1, 5, 3, 6, 2, 4)
        return k.reshape(sh + (pg, hd)).float(), v.reshape(sh + (pg, hd)).float()
    e = pg * hd
    kq, ks, vq, vs = x.split([e, 2 * pg * n, e, 2 * pg * n], dim=1)
    k = kq.contiguous().view(torch.int8).view(N, pg // 16, hd // 64, 4, 16, 2, 8).permute(0, 1, 4, 2, 5, 3, 6)
    v = vq.contiguous().view(torch.int8).view(N, pg // 32, n, 4, 16, 2, 2, 4).permute(0, 1, 6, 3, 7, 2, 5, 4)
    ks = ks.contiguous().view(torch.float16).view(N, pg // 16, 4, n, 4).permute(0, 1, 2, 4, 3)
    vs = vs.contiguous().view(torch.float16).view(N, pg // 32, 4, n, 2, 4).permute(0, 1, 4, 2, 5, 3)
    k = k.reshape(N, pg, n, 32).float() * ks.reshape(N, pg, n, 1).float()
    v = v.reshape(N, pg, n, 32).float() * vs.reshape(N, pg, n, 1).float()
    return k.reshape(sh + (pg, hd)), v.reshape(sh + (pg, hd))


# ------------------------------------------------------------------- inputs

def _gen(seed, *more):
    g = torch.Generator(device=DEV)
    v = 1469598103934665603
    for m in (seed,) + more:
        v = ((v ^ (int(m) & 0xffffffff)) * 1099511628211) & 0x7fffffffffffffff
    g.manual_seed(v)
    return g


def _pages(c, n, g):
    """Random pages: elements of about unit size, keys with a mean of their own per page and dim, as keys that a
    rotation has passed over have."""
    kv, pg, hd = c["kv"], c["page"], c["hd"]
    p, d = torch.arange(pg, device=DEV)[:, None], torch.arange(hd, device=DEV)
    if c["t"] == "f16":
        raw = torch.randn(n * kv, _block_bytes(c) // 2, device=DEV, generator=g, dtype=torch.float16)
        at = _k_at(c, p, d).reshape(-1)
        k = raw[:, at].view(n * kv, pg, hd)
        raw[:, at] = (0.7 * k + torch.randn(n * kv, 1, hd, device=DEV, generator=g, dtype=torch.float16)).view(n * kv, -1)
        return raw.view(torch.uint8).view(-1)
    raw = torch.randint(-(1 << 31), (1 << 31) - 1, (n * kv, _block_bytes(c) // 4), dtype=torch.int32, device=DEV, generator=g)
    raw = raw.view(torch.uint8).view(n * kv, _block_bytes(c))
    e, s = pg * hd, pg * (hd // 32)
    for at in (e, 2 * e + 2 * s):  # scales: -127..127 stand for about -1.7..1.7
        z = (torch.rand(raw.shape[0], s, device=DEV, generator=g) * 0.012 + 0.008).to(torch.float16)
        raw[:, at:at + 2 * s] = z.view(torch.uint8).view(raw.shape[0], 2 * s)
    for at in (0, e + 2 * s):  # -128 is not a quant of the store
        q = raw[:, at:at + e]
        q[q == 128] = 129
    at = _k_at(c, p, d).reshape(-1)
    k = raw[:, at].view(torch.int8).view(n * kv, pg, hd).float()
    m = torch.randn(n * kv, 1, hd, device=DEV, generator=g) * 40.0
    raw[:, at] = (0.5 * k + m).round().clamp(-127, 127).to(torch.int8).view(n * kv, -1).view(torch.uint8)
    return raw.view(-1)


def _sample_inputs(c, seed):
    g, n, V = _gen(seed, 2), c["rows"], c["vocab"]
    x = torch.randn(n, V, device=DEV, generator=g) * 2.0
    if c["peak"]:  # a few likely tokens, the next ones less and less so
        r = torch.argsort(torch.rand(n, V, device=DEV, generator=g), dim=1)[:, :min(V, 48)]
        up = c["peak"] - 1.5 * torch.log1p(torch.arange(r.shape[1], device=DEV, dtype=torch.float32))
        x.scatter_add_(1, r, (up + torch.randn(n, r.shape[1], device=DEV, generator=g)).clamp_min_(0.0))
    s = dict(case=c, logits=x, u=torch.rand(n, device=DEV, generator=g))
    if c["how"] == "mixed":
        rs = np.random.RandomState(seed & 0x7fffffff)
        temp = rs.choice([0.0, 0.2, 0.7, 1.0, 1.4], n)
        k = rs.choice([0, 0, 1, 20, 40, 100], n)
        p = rs.choice([1.0, 0.95, 0.9, 0.5], n)
        m = rs.choice([0.0, 0.0, 0.05, 0.1], n)
    else:
        temp, k, p, m = (np.full(n, c[i]) for i in ("temp", "k", "p", "m"))
    for name, v, t, off in (("temp", temp, np.float32, 1.0), ("k", k, np.int32, 0), ("p", p, np.float32, 1.0), ("m", m, np.float32, 0.0)):
        s[name] = None if c["how"] == "one" and c[name] == off else torch.from_numpy(v.astype(t)).to(DEV)
    return s


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "sample":
        return _sample_inputs(c, seed)
    g, rs = _gen(seed, 1), np.random.RandomState(seed & 0x7fffffff)
    lens, rows = np.array(_lens(c)), np.array(_rows(c))
    s = dict(case=c)
    common = np.zeros(len(lens), int)
    if c["kind"] == "shared":
        s["group_pages"] = torch.tensor(_shared_pages(c), dtype=torch.int32, device=DEV)
        s["group_start"] = torch.arange(c["groups"] + 1, dtype=torch.int32, device=DEV) * c["members"]
        common[:c["groups"] * c["members"]] = np.repeat(_shared_pages(c), c["members"])
    else:
        order = rs.permutation(len(lens))
        lens, rows = lens[order], rows[order]
    need = -(-lens // c["page"])
    table, n = np.zeros((len(lens), int(need.max())), int), 0
    for b, m in enumerate(need):
        k = int(common[b]) if c["kind"] == "shared" and b % c["members"] else 0  # the first member's pages
        table[b, :k] = table[b - b % c["members"], :k] if k else 0
        table[b, k:m] = np.arange(n, n + m - k)
        n += int(m) - k
    n += 3
    table = rs.permutation(n)[table]
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    s |= dict(pages=_pages(c, n, g), table=torch.from_numpy(table.astype(np.int32)).to(DEV), n_pages=n, s_rows=int(start[-1]),
              seq_len=torch.from_numpy(lens.astype(np.int32)).to(DEV), row_start=torch.from_numpy(start).to(DEV) if max(rows) > 1 else None)
    if c["kind"] == "bounds":
        s["bounds"] = torch.zeros(n, c["kv"], 2, c["hd"], dtype=torch.float16, device=DEV)
        return s
    s["q"] = torch.randn(s["s_rows"], c["heads"] * c["hd"], device=DEV, generator=g)
    if c["kind"] == "selected":  # kept beside the cache: of whole pages, and of the sequences' last ones what they hold
        s["bounds"] = torch.zeros(n, c["kv"], 2, c["hd"], dtype=torch.float16, device=DEV)
        for i in range(0, n, 512):
            k, _ = _blocks(s, torch.arange(i, min(n, i + 512), device=DEV))
            s["bounds"][i:i + 512] = torch.stack([k.amin(2), k.amax(2)], 2).half()
        last = s["table"].long().gather(1, (s["seq_len"].long()[:, None] - 1) // c["page"])[:, 0]
        s["bounds"][last] = _bounds_of(s, last, (s["seq_len"].long() - 1) % c["page"] + 1)
    return s


# -------------------------------------------------------------------- passes

def _bounds_of(s, ids, count):
    """Bounds [n, kv, 2, hd] of the first count [n] positions of the pages ids [n]."""
    k, _ = _blocks(s, ids)
    gone = (torch.arange(s["case"]["page"], device=DEV)[None] >= count[:, None])[:, None, :, None]
    return torch.stack([k.masked_fill(gone, math.inf).amin(2), k.masked_fill(gone, -math.inf).amax(2)], 2).half()


def _plain_sample(s):
    x = s["logits"].double()  # sums over many tokens, and their borders
    n, V = x.shape
    one = torch.ones(n, 1, dtype=torch.float64, device=DEV)
    temp = one if s["temp"] is None else s["temp"].double()[:, None]
    w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(temp > 0, temp, one))
    order = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices
    y = w.gather(1, order)
    if s["k"] is not None:
        k = s["k"].long()[:, None]
        y = torch.where(torch.arange(V, device=DEV)[None] < torch.where((k <= 0) | (k > V), V, k), y, 0.0)
    if s["p"] is not None:
        before = torch.cumsum(y, 1) - y
        y = torch.where((before < s["p"].double()[:, None] * y.sum(1, keepdim=True)) | (s["p"][:, None] >= 1), y, 0.0)
    if s["m"] is not None:
        y = torch.where(y >= s["m"].double()[:, None], y, 0.0)
    y = torch.where((temp <= 0) & (torch.arange(V, device=DEV)[None] > 0), 0.0, y)
    kept = torch.zeros_like(w).scatter_(1, order, y)
    run_, total = torch.cumsum(kept, 1), kept.sum(1, keepdim=True)
    i = (run_ <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp_max_(V - 1)
    return dict(ids=i[:, 0].int(), p=(kept.gather(1, i) / total)[:, 0].float())


def _where(s):
    """Sequence and position of every row."""
    n = s["seq_len"].long()
    if s["row_start"] is None:
        return torch.arange(s["s_rows"], device=DEV), n - 1
    st = s["row_start"].long()
    b = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), st[1:] - st[:-1], output_size=s["s_rows"])
    return b, n[b] - (st[1:] - st[:-1])[b] + torch.arange(s["s_rows"], device=DEV) - st[b]


def _plain_select(s, b, pos):
    """Pages [S, kv, P] that the rows at `pos` of sequences b see, of the table's columns."""
    c, S = s["case"], s["s_rows"]
    P, G = s["table"].shape[1], c["heads"] // c["kv"]
    q = s["q"].view(S, c["kv"], G, c["hd"]).double()  # two pages' scores may lie next to each other
    q = torch.cat([q.clamp_max(0.0).sum(2), q.clamp_min(0.0).sum(2)], 2)  # [S, kv, 2 hd]: lo takes the negative parts
    x = torch.zeros(S, c["kv"], P, dtype=torch.float64, device=DEV)
    if s["row_start"] is None or s["seq_len"].numel() > 1:
        R = max(_rows(c))
        i = torch.zeros_like(b) if s["row_start"] is None else torch.arange(S, device=DEV) - s["row_start"].long()[b]
        y = torch.zeros(s["seq_len"].numel(), R, c["kv"], 2 * c["hd"], dtype=torch.float64, device=DEV)
        y[b, i] = q
        e = s["bounds"][s["table"].long()].view(-1, P, c["kv"], 2 * c["hd"]).double()  # [B, P, kv, 2 hd]
        x = torch.matmul(y.permute(0, 2, 1, 3), e.permute(0, 2, 3, 1).contiguous()).permute(0, 2, 1, 3)[b, i]
    else:
        e = s["bounds"][s["table"][0].long()].view(P, c["kv"], 2 * c["hd"]).double()
        x = torch.matmul(q.transpose(0, 1), e.permute(1, 2, 0).contiguous()).transpose(0, 1)
    col, mine = torch.arange(P, device=DEV)[None, None], (pos // c["page"])[:, None, None]
    x = x.masked_fill((col == mine) | (col < c["first"]), math.inf).masked_fill(col > mine, -math.inf)
    order = torch.sort(x, dim=2, descending=True, stable=True).indices[:, :, :c["select"]]
    return torch.zeros(S, c["kv"], P, dtype=torch.bool, device=DEV).scatter_(2, order, True) & (col <= mine)


def _plain_attn(s):
    c = s["case"]
    nh, kv, hd, (B, P) = c["heads"], c["kv"], c["hd"], s["table"].shape
    G = nh // kv
    b, pos = _where(s)
    k, v = (x.transpose(1, 2).reshape(B, kv, P * c["page"], hd) for x in _blocks(s, s["table"].long()))
    L = P * c["page"]
    if s["row_start"] is None:
        R, i = 1, torch.zeros_like(b)
    else:
        R, i = max(_rows(c)), torch.arange(s["s_rows"], device=DEV) - s["row_start"].long()[b]
    q = torch.zeros(B, R, nh * hd, device=DEV)
    at = torch.full((B, R), -1, device=DEV, dtype=torch.long)
    q[b, i], at[b, i] = s["q"], pos
    q = q.view(B, R, kv, G, hd).permute(0, 2, 4, 1, 3).reshape(B, kv, hd, R * G)
    x = torch.matmul(k, q) * (1.0 / math.sqrt(hd))  # [B, kv, L, R G]
    seen = (torch.arange(L, device=DEV)[None, :, None] <= at[:, None, :])[:, None]  # [B, 1, L, R]
    if c["kind"] == "selected":
        m = torch.zeros(B, R, kv, P, dtype=torch.bool, device=DEV)
        m[b, i] = _plain_select(s, b, pos)
        seen = seen & m.permute(0, 2, 3, 1).repeat_interleave(c["page"], dim=2)  # [B, kv, L, R]
    x = x.view(B, kv, L, R, G).masked_fill_(~seen[..., None], -math.inf)
    m = x.amax(dim=2, keepdim=True).clamp_min_(-3.0e38)
    w = x.sub_(m).exp_()
    l = w.sum(dim=2)  # [B, kv, R, G]
    o = torch.matmul(w.view(B, kv, L, R * G).transpose(2, 3).contiguous(), v).view(B, kv, R, G, hd) / l[..., None]
    return o.permute(0, 2, 1, 3, 4).reshape(B, R, nh * hd)[b, i]


def _plain_bounds(s):
    pg, n = s["case"]["page"], s["seq_len"].long()
    rows = torch.ones_like(n) if s["row_start"] is None else (s["row_start"][1:] - s["row_start"][:-1]).long()
    col = torch.arange(s["table"].shape[1], device=DEV)[None]
    b, j = torch.nonzero((col >= (n - rows)[:, None] // pg) & (col * pg < n[:, None]), as_tuple=True)
    ids = s["table"][b, j].long()
    s["bounds"][ids] = _bounds_of(s, ids, n[b] - j * pg)
    return s["bounds"]


_ctx = None


def _context():
    """One context for all passes, as a program has it."""
    global _ctx
    if _ctx is None:
        from kestrel_amd import kmoe

        _ctx = kmoe.Context(0)
    return _ctx


def run(s):
    c = s["case"]
    if not own:
        return _plain_sample(s) if c["kind"] == "sample" else _plain_bounds(s) if c["kind"] == "bounds" else _plain_attn(s)
    ctx = _context()
    if c["kind"] == "sample":
        p = torch.empty(c["rows"], device=DEV)
        ids = ctx.sample(s["logits"], s["u"], temperature=s["temp"], top_k=s["k"], top_p=s["p"], min_p=s["m"], prob=p)
        return dict(ids=ids, p=p)
    from kestrel_amd.kmoe import F16, Q8_0, PagedKV

    kv = PagedKV(F16 if c["t"] == "f16" else Q8_0, c["kv"], c["hd"], c["page"])
    batch = ctx.paged_batch(s["table"], s["seq_len"], s["row_start"], s["s_rows"])
    if c["kind"] == "bounds":
        return ctx.paged_bounds(kv, s["pages"], batch, s["bounds"])
    if c["kind"] == "selected":
        return ctx.paged_attention_selected(kv, s["pages"], s["bounds"], batch, s["q"], c["heads"], c["select"], n_first=c["first"])
    return ctx.paged_attention_shared(kv, s["pages"], batch, ctx.paged_groups(s["group_start"], s["group_pages"]), s["q"], c["heads"])


def work(case):
    c = case
    if c["kind"] == "sample":  # the logits once; an exponential (of some ten operations) and a sum each
        return dict(bytes=c["rows"] * (4 * c["vocab"] + 8), flops=12 * c["rows"] * c["vocab"])
    per = c["hd"] * 2 if c["t"] == "f16" else c["hd"] // 32 * 34  # one position of one kv head, K or V
    lens, rows, pg = _lens(c), _rows(c), c["page"]
    S, edge = sum(rows), 4 * c["kv"] * c["hd"]  # edge: a page's bounds
    if c["kind"] == "bounds":
        pages = [(n - r) // pg for n, r in zip(lens, rows)]
        seen = sum(n - a * pg for n, a in zip(lens, pages))
        return dict(bytes=seen * c["kv"] * per + edge * sum(-(-n // pg) - a for n, a in zip(lens, pages)), flops=2 * seen * c["kv"] * c["hd"])
    io = S * c["heads"] * c["hd"] * 8
    if c["kind"] == "shared":
        pairs = sum(sum(range(n - r + 1, n + 1)) for n, r in zip(lens, rows))
        once = sum(lens) - sum((c["members"] - 1) * n * pg for n in _shared_pages(c))
        return dict(bytes=once * c["kv"] * 2 * per + io, flops=4 * pairs * c["heads"] * c["hd"])
    bytes_, flops = io, 0
    for n, r in zip(lens, rows):  # rows of a chunk may select the same pages: those of one row at least are read
        pages = -(-n // pg)
        bytes_ += pages * edge + min(c["select"], pages) * pg * c["kv"] * 2 * per
        seen = min(c["select"], pages) * pg * r
        flops += 4 * seen * c["heads"] * c["hd"] + 4 * r * pages * c["kv"] * c["hd"]
    return dict(bytes=bytes_, flops=flops)


# ------------------------------------------------------------------ 64 bits

def _element(s, base, p, at, sat):
    """Elements [kv, positions, hd] in 64 bits by their places in the pages; base [positions] the pages' ids, p the positions in them."""
    c = s["case"]
    h = torch.arange(c["kv"], device=DEV)[:, None, None]
    o = (base[None, :, None] * c["kv"] + h) * _block_bytes(c)
    d = torch.arange(c["hd"], device=DEV)
    i = at(c, p[None, :, None], d)
    if c["t"] == "f16":
        return s["pages"].view(torch.float16)[o // 2 + i].double()
    j = o + sat(c, p[None, :, None], d // 32)
    return s["pages"].view(torch.int8)[o + i].double() * s["pages"].view(torch.float16)[j // 2].double()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "sample":
        x, u = s["logits"].cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
        temp, k, p, m = (np.full(c["rows"], off) if s[n] is None else s[n].cpu().numpy().astype(np.float64)
                         for n, off in (("temp", 1.0), ("k", 0), ("p", 1.0), ("m", 0.0)))
        ids, prob = np.zeros(c["rows"], np.int32), np.ones(c["rows"])
        for r in range(c["rows"]):
            if temp[r] <= 0:
                ids[r] = int(np.argmax(x[r]))
                continue
            w = np.exp((x[r] - x[r].max()) / temp[r])
            kept = np.lexsort((np.arange(c["vocab"]), -x[r])) if k[r] > 0 or p[r] < 1 else np.arange(c["vocab"])
            if 0 < k[r]:
                kept = kept[:int(k[r])]
            if p[r] < 1:
                held = np.cumsum(w[kept])
                kept = kept[:int(np.searchsorted(held, p[r] * held[-1])) + 1]
            kept = np.sort(kept[w[kept] >= m[r]])
            held = np.cumsum(w[kept])
            ids[r] = kept[min(int(np.searchsorted(held, u[r] * held[-1], side="right")), kept.size - 1)]
            prob[r] = w[ids[r]] / held[-1]
        return dict(ids=torch.from_numpy(ids).to(DEV), p=torch.from_numpy(prob).to(DEV))
    nh, kv, hd, pg = c["heads"], c["kv"], c["hd"], c["page"]
    lens = s["seq_len"].tolist()
    start = s["row_start"].tolist() if s["row_start"] is not None else list(range(len(lens) + 1))
    if c["kind"] == "bounds":
        for b, n in enumerate(lens):
            for j in range((n - (start[b + 1] - start[b])) // pg, -(-n // pg)):
                p = torch.arange(min(pg, n - j * pg), device=DEV)
                k = _element(s, s["table"][b, j].long().expand(p.numel()), p, _k_at, _ks_at)
                s["bounds"][s["table"][b, j]] = torch.stack([k.min(1).values, k.max(1).values], 1).half()
        return s["bounds"].double()
    out = []
    for b, n in enumerate(lens):
        r = start[b + 1] - start[b]
        p = torch.arange(n, device=DEV)
        base = s["table"][b].long()[p // pg]
        k, v = _element(s, base, p % pg, _k_at, _ks_at), _element(s, base, p % pg, _v_at, _vs_at)
        q = s["q"][start[b]:start[b + 1]].double().view(r, kv, nh // kv, hd).permute(1, 2, 0, 3)  # [kv, G, r, hd]
        e = s["bounds"][s["table"][b].long()[:-(-n // pg)]].double() if c["kind"] == "selected" else None  # [P, kv, 2, hd]
        o = torch.empty(kv, nh // kv, r, hd, dtype=torch.float64, device=DEV)
        step = 16 if e is not None else 256
        for i in range(0, r, step):  # rows at a time
            at = torch.arange(n - r + i, min(n, n - r + i + step), device=DEV)
            x = torch.matmul(q[:, :, i:i + step].reshape(kv, -1, hd), k.transpose(1, 2).contiguous()).view(kv, nh // kv, -1, n) / hd ** 0.5
            hide = (p[None] > at[:, None])[None, None]
            if e is not None:
                best = torch.zeros(kv, at.numel(), e.shape[0], dtype=torch.float64, device=DEV)
                for h in range(nh // kv):
                    y = q[:, h, i:i + step, None, :]  # [kv, rows, 1, hd]
                    best += torch.maximum(y * e[:, :, 0].transpose(0, 1)[:, None], y * e[:, :, 1].transpose(0, 1)[:, None]).sum(-1)
                col, mine = torch.arange(e.shape[0], device=DEV)[None, None], (at // pg)[None, :, None]
                always = (col == mine) | (col < c["first"])
                rank = torch.argsort(torch.argsort(torch.where(always, math.inf, torch.where(col < mine, best, -math.inf)), dim=2, descending=True, stable=True), dim=2)
                hide = hide | ~((rank < c["select"]) & (col <= mine))[:, None, :, (p // pg)]
            w = torch.softmax(x.masked_fill(hide, -math.inf), dim=-1)
            o[:, :, i:i + step] = torch.matmul(w.reshape(kv, -1, n), v).view(kv, nh // kv, -1, hd)
        out.append(o.permute(2, 0, 1, 3).reshape(r, nh * hd))
    return torch.cat(out)
