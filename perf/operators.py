"""Timed cases of the paged key-value cache: the cache store and its read-back,
attention over the pages (one token per sequence, prompt chunks, both in one
batch; a sliding window with visible first positions), and page copies.

listed() names the cases, draw() gives more of the same ranges, prepare() makes
what a program that serves many sequences holds before the call (pages in HBM,
page table, lengths, the rows), run() is one pass, work() the bytes and
operations it cannot do without, exact() the same outputs in 64 bits.

With `own` false run() takes elementary torch operations, with `own` true the
calls of kestrel_amd.kmoe.Context.

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
        # the smallest call: one sequence that has just begun, one new token
        dict(name="decode-1-at-37", kind="attn", t="f16", heads=16, kv=4, hd=128, page=64, seqs=1, lo=37, hi=37,
             prompts=0, rows=1, window=0, sink=0),
        # one sequence over a very long context
        dict(name="decode-1-at-131000", kind="attn", t="f16", heads=32, kv=8, hd=128, page=256, seqs=1, lo=131000,
             hi=131000, prompts=0, rows=1, window=0, sink=0),
        # a decode step of 64 sequences of very different lengths
        dict(name="decode-64-ragged", kind="attn", t="f16", heads=32, kv=8, hd=128, page=64, seqs=64, lo=100, hi=8192,
             prompts=0, rows=1, window=0, sink=0),
        # many short sequences over an 8-bit cache, heads of 64
        dict(name="decode-200-q8", kind="attn", t="q8_0", heads=16, kv=8, hd=64, page=32, seqs=200, lo=30, hi=4096,
             prompts=0, rows=1, window=0, sink=0),
        # a decode step of long chats that keep a window and their first positions
        dict(name="window-48", kind="attn", t="f16", heads=16, kv=4, hd=128, page=64, seqs=48, lo=900, hi=20000,
             prompts=0, rows=1, window=1024, sink=4),
        # a whole prompt
        dict(name="prompt-1777", kind="attn", t="f16", heads=16, kv=4, hd=128, page=64, seqs=1, lo=1777, hi=1777,
             prompts=1, rows=1777, window=0, sink=0),
        # decoding sequences and two prompt chunks in one batch, 8-bit cache
        dict(name="mixed-9-q8", kind="attn", t="q8_0", heads=32, kv=8, hd=128, page=64, seqs=9, lo=50, hi=6000,
             prompts=2, rows=512, window=0, sink=0),
        # a prompt chunk of a long document under the window
        dict(name="window-prompt-2048", kind="attn", t="f16", heads=32, kv=8, hd=128, page=64, seqs=1, lo=8100, hi=8100,
             prompts=1, rows=2048, window=1024, sink=4),
        # a decode step's new rows into the cache, RoPE on the way
        dict(name="store-64", kind="store", t="f16", heads=32, kv=8, hd=128, page=64, seqs=64, lo=100, hi=8192,
             prompts=0, rows=1, neox=1),
        # a prompt's rows into an 8-bit cache
        dict(name="store-1777-q8", kind="store", t="q8_0", heads=16, kv=4, hd=128, page=64, seqs=1, lo=1777, hi=1777,
             prompts=1, rows=1777, neox=0),
        # the one shared page of a forked sequence that is about to be written
        dict(name="copy-fork-q8", kind="copy", t="q8_0", kv=4, hd=128, page=64, layers=24, pool=64, n=1),
        # compaction: the last pages of a fragmented pool move to its front
        dict(name="copy-compact", kind="copy", t="f16", kv=4, hd=128, page=64, layers=24, pool=330, n=150),
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _padded(c):
    """Elements of K over all sequences, each at the longest one's length."""
    return c["seqs"] * c["hi"] * c["kv"] * c["hd"]


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "attn", "store", "store", "copy"])
    t, page = rng.choice(["f16", "f16", "q8_0"]), rng.choice([32, 64, 128, 256])
    heads, kv, hd = rng.choice([(16, 4, 128), (32, 8, 128), (16, 16, 128), (16, 8, 64), (12, 4, 64), (14, 2, 64),
                                (24, 8, 128), (32, 2, 128)])
    if kind == "copy":
        layers, n = _between(rng, 1, 32), _between(rng, 1, 400)
        c = dict(kind="copy", t=t, kv=kv, hd=hd, page=page, layers=layers, pool=2 * n + rng.randint(1, 40), n=n)
        while c["pool"] * c["layers"] * _page_bytes(c) > 1 << 30 and c["n"] > 1:
            c["n"] = c["n"] // 2
            c["pool"] = 2 * c["n"] + rng.randint(1, 40)
        return c
    form = rng.choice(["decode", "decode", "prompt", "mixed"])
    seqs = 1 if rng.random() < 0.2 else _between(rng, 1, 256) if form == "decode" else _between(rng, 1, 24)
    if kind == "store":
        c = dict(kind="store", t=t, heads=heads, kv=kv, hd=hd, page=page, seqs=seqs, lo=1, hi=_between(rng, 2, 8192),
                 prompts=0, rows=1, neox=rng.randint(0, 1))
    else:
        c = dict(kind="attn", t=t, heads=heads, kv=kv, hd=hd, page=page, seqs=seqs, lo=1, hi=_between(rng, 2, 65536),
                 prompts=0, rows=1, window=0, sink=0)
        if rng.random() < 0.35:
            c["window"], c["sink"] = _between(rng, 1, 4096), rng.choice([0, 1, 4, 37])
    c["lo"] = _between(rng, 1, c["hi"])
    if form != "decode":
        c["prompts"] = seqs if form == "prompt" else rng.randint(1, seqs)
        c["rows"] = _between(rng, 2, 2048)
    # at most what the largest listed case takes, and what pads to a few GB in 32 bits
    while (_cost(c) > _cost(max(listed(), key=_cost)) or _padded(c) > 1 << 29
           or (c["prompts"] and _padded(c) * min(c["rows"], c["hi"]) * heads // (kv * hd) > 1 << 29)):
        if c["seqs"] > 1 and rng.random() < 0.5:
            c["seqs"] = max(1, c["seqs"] // 2)
            c["prompts"] = min(c["prompts"], c["seqs"])
        else:
            c["hi"] = max(2, c["hi"] // 2)
            c["lo"] = min(c["lo"], c["hi"])
    return c


def _lens(c):
    """The sequences' lengths, spread evenly over the logarithm of lo..hi, shortest first."""
    if c["seqs"] == 1:
        return [c["hi"]]
    a, b = math.log(c["lo"]), math.log(c["hi"])
    return [min(c["hi"], max(c["lo"], int(round(math.exp(a + (b - a) * i / (c["seqs"] - 1)))))) for i in range(c["seqs"])]


def _rows(c):
    """New rows of each sequence: chunks of `rows` for the longest ones, one for the others."""
    n = _lens(c)
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


# ------------------------------------------------------------------- inputs

def _gen(seed, *more):
    g = torch.Generator(device=DEV)
    v = 1469598103934665603
    for m in (seed,) + more:
        v = ((v ^ (int(m) & 0xffffffff)) * 1099511628211) & 0x7fffffffffffffff
    g.manual_seed(v)
    return g


def _pages(c, n, g, layers=1):
    """Random pages: elements of about unit size."""
    nb = layers * n * _page_bytes(c)
    if c["t"] == "f16":
        return torch.randn(nb // 2, device=DEV, generator=g, dtype=torch.float16).view(torch.uint8)
    raw = torch.randint(-(1 << 31), (1 << 31) - 1, (nb // 4,), dtype=torch.int32, device=DEV, generator=g).view(torch.uint8)
    raw = raw.view(layers * n * c["kv"], _block_bytes(c))
    e, s = c["page"] * c["hd"], c["page"] * (c["hd"] // 32)
    for at in (e, 2 * e + 2 * s):  # scales: -127..127 stand for about -1.7..1.7
        d = (torch.rand(raw.shape[0], s, device=DEV, generator=g) * 0.012 + 0.008).to(torch.float16)
        raw[:, at:at + 2 * s] = d.view(torch.uint8).view(raw.shape[0], 2 * s)
    raw.view(-1).view(torch.int8)  # -128 is not a quant of the store
    for at in (0, e + 2 * s):
        q = raw[:, at:at + e]
        q[q == 128] = 129
    return raw.view(-1)


def prepare(case, seed):
    c, g = dict(case), _gen(seed, 1)
    if c["kind"] == "copy":
        ids = torch.from_numpy(np.random.RandomState(seed & 0x7fffffff).permutation(c["pool"]).astype(np.int64))
        src, dst = ids[:c["n"]], ids[c["n"]:2 * c["n"]]
        pool = _pages(c, c["pool"], g, c["layers"]).view(torch.int32).view(c["layers"], c["pool"], -1)
        return dict(case=c, pool=pool, src=src.tolist(), dst=dst.tolist())
    rs = np.random.RandomState(seed & 0x7fffffff)
    order = rs.permutation(c["seqs"])
    lens, rows = np.array(_lens(c))[order], np.array(_rows(c))[order]
    cols = int(-(-max(lens) // c["page"]))
    need = -(-lens // c["page"])
    n = int(need.sum()) + 3
    ids, table, at = rs.permutation(n), np.zeros((c["seqs"], cols), np.int32), 0
    for b in range(c["seqs"]):
        table[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    s = dict(case=c, pages=_pages(c, n, g), table=torch.from_numpy(table).to(DEV),
             seq_len=torch.from_numpy(lens.astype(np.int32)).to(DEV), n_pages=n, s_rows=int(start[-1]),
             row_start=torch.from_numpy(start).to(DEV) if c["prompts"] else None)
    S, nh, kv, hd = s["s_rows"], c["heads"], c["kv"], c["hd"]
    if c["kind"] == "attn":
        s["q"] = torch.randn(S, nh * hd, device=DEV, generator=g)
    else:
        s["qkv"] = torch.randn(S, (nh + 2 * kv) * hd, device=DEV, generator=g)
        e = (-(2.0 * np.arange(hd // 2, dtype=np.float32)) / np.float32(hd)).astype(np.float32)
        s["inv_freq"] = torch.from_numpy(np.power(np.float32(10000.0), e, dtype=np.float32)).to(DEV)
    return s


# -------------------------------------------------------------------- passes

def _where(s):
    """Sequence and position of every row."""
    n = s["seq_len"].long()
    if s["row_start"] is None:
        return torch.arange(s["s_rows"], device=DEV), n - 1
    st = s["row_start"].long()
    b = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), st[1:] - st[:-1], output_size=s["s_rows"])
    return b, n[b] - (st[1:] - st[:-1])[b] + torch.arange(s["s_rows"], device=DEV) - st[b]


def _unpaged(s):
    """K and V of every sequence [seqs, kv, positions, hd] in 32 bits, from the pages of its table."""
    c = s["case"]
    B, P = s["table"].shape
    kv, hd, pg = c["kv"], c["hd"], c["page"]
    x = s["pages"].view(s["n_pages"], kv, _block_bytes(c))[s["table"].long()]  # [B, P, kv, bytes]
    if c["t"] == "f16":
        x = x.view(torch.float16)
        k = x[..., :pg * hd].reshape(B, P, kv, pg // 16, hd // 32, 4, 16, 8).permute(0, 2, 1, 3, 6, 4, 5, 7)
        v = x[..., pg * hd:].reshape(B, P, kv, pg // 32, hd // 16, 4, 16, 2, 4).permute(0, 2, 1, 3, 7, 5, 8, 4, 6)
        return k.reshape(B, kv, P * pg, hd).float(), v.reshape(B, kv, P * pg, hd).float()
    e, n = pg * hd, hd // 32
    kq, ks, vq, vs = x.split([e, 2 * pg * n, e, 2 * pg * n], dim=-1)
    k = kq.contiguous().view(torch.int8).reshape(B, P, kv, pg // 16, hd // 64, 4, 16, 2, 8).permute(0, 2, 1, 3, 6, 4, 7, 5, 8)
    v = vq.contiguous().view(torch.int8).reshape(B, P, kv, pg // 32, n, 4, 16, 2, 2, 4).permute(0, 2, 1, 3, 8, 5, 9, 4, 7, 6)
    ks = ks.contiguous().view(torch.float16).reshape(B, P, kv, pg // 16, 4, n, 4).permute(0, 2, 1, 3, 4, 6, 5)
    vs = vs.contiguous().view(torch.float16).reshape(B, P, kv, pg // 32, 4, n, 2, 4).permute(0, 2, 1, 3, 6, 4, 7, 5)
    k = k.reshape(B, kv, P * pg, n, 32).float() * ks.reshape(B, kv, P * pg, n, 1).float()
    v = v.reshape(B, kv, P * pg, n, 32).float() * vs.reshape(B, kv, P * pg, n, 1).float()
    return k.reshape(B, kv, P * pg, hd), v.reshape(B, kv, P * pg, hd)


def _plain_attn(s):
    c = s["case"]
    nh, kv, hd, B = c["heads"], c["kv"], c["hd"], s["table"].shape[0]
    G = nh // kv
    b, pos = _where(s)
    k, v = _unpaged(s)
    L = k.shape[2]
    if s["row_start"] is None:
        R, i = 1, torch.zeros_like(b)
    else:
        st = s["row_start"].long()
        R, i = max(_rows(c)), torch.arange(s["s_rows"], device=DEV) - st[b]
    q = torch.zeros(B, R, nh * hd, device=DEV)
    at = torch.full((B, R), -1, device=DEV, dtype=torch.long)
    q[b, i], at[b, i] = s["q"], pos
    q = q.view(B, R, kv, G, hd).permute(0, 2, 4, 1, 3).reshape(B, kv, hd, R * G)
    x = torch.matmul(k, q) * (1.0 / math.sqrt(hd))  # [B, kv, L, R G]
    p, at = torch.arange(L, device=DEV)[None, :, None], at[:, None, :]
    seen = p <= at
    if c["window"]:
        seen = seen & ((p > at - c["window"]) | (p < c["sink"]))
    x = x.view(B, kv, L, R, G).masked_fill_(~seen[:, None, :, :, None], -math.inf)
    m = x.amax(dim=2, keepdim=True).clamp_min_(-3.0e38)
    w = x.sub_(m).exp_()
    l = w.sum(dim=2)  # [B, kv, R, G]
    o = torch.matmul(w.view(B, kv, L, R * G).transpose(2, 3).contiguous(), v).view(B, kv, R, G, hd) / l[..., None]
    return o.permute(0, 2, 1, 3, 4).reshape(B, R, nh * hd)[b, i]


def _rotated(x, ang, neox):
    """x [S, heads, hd] rotated by ang [S, hd / 2], whole heads."""
    cs, sn = torch.cos(ang).to(x.dtype)[:, None, :], torch.sin(ang).to(x.dtype)[:, None, :]
    h = x.shape[-1] // 2
    a, b = (x[..., :h], x[..., h:]) if neox else (x[..., 0::2], x[..., 1::2])
    u, w = a * cs - b * sn, a * sn + b * cs
    return torch.cat([u, w], -1) if neox else torch.stack([u, w], -1).flatten(-2)


def _plain_store(s):
    c = s["case"]
    S, nh, kv, hd, pg = s["s_rows"], c["heads"], c["kv"], c["hd"], c["page"]
    b, pos = _where(s)
    q, k, v = s["qkv"].view(S, nh + 2 * kv, hd).split([nh, kv, kv], dim=1)
    ang = (pos.float()[:, None] * s["inv_freq"]).double()  # the angle is the 32-bit product, as in the framework's other RoPE calls
    q, k = _rotated(q, ang, c["neox"]), _rotated(k, ang, c["neox"])
    p, d, h = (pos % pg)[:, None, None], torch.arange(hd, device=DEV), torch.arange(kv, device=DEV)[:, None]
    base = (s["table"][b, pos // pg].long()[:, None, None] * kv + h) * _block_bytes(c)  # [S, kv, 1]
    got = []
    if c["t"] == "f16":
        flat = s["pages"].view(torch.float16)
        for x, at in ((k, _k_at), (v, _v_at)):
            i = base // 2 + at(c, p, d)
            flat[i] = x.half()
            got.append(flat[i].reshape(S, kv * hd))
    else:
        flat, u = s["pages"], torch.arange(hd // 32, device=DEV)
        for x, at, sat in ((k, _k_at, _ks_at), (v, _v_at, _vs_at)):
            x = x.reshape(S, kv, hd // 32, 32).double()
            scale = (x.abs().amax(-1) / 127.0).half()
            z = scale.double()[..., None]
            n = torch.where(z > 0, x / z, torch.zeros_like(x)).round().clamp(-127, 127).to(torch.int8)
            i, j = base + at(c, p, d), (base + sat(c, p, u))[..., None] + torch.arange(2, device=DEV)
            flat[i] = n.view(torch.uint8).reshape(S, kv, hd)
            flat[j] = scale.view(torch.uint8).reshape(S, kv, hd // 32, 2)
            y = flat[i].view(torch.int8).reshape(S, kv, hd // 32, 32).float() * flat[j].view(torch.float16).float()
            got.append(y.half().reshape(S, kv * hd))
    return dict(q=q.reshape(S, nh * hd), k=got[0], v=got[1])


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
        if c["kind"] == "attn":
            return _plain_attn(s)
        if c["kind"] == "store":
            return _plain_store(s)
        s["pool"][:, s["dst"]] = s["pool"][:, s["src"]]
        return s["pool"]
    ctx = _context()
    from kestrel_amd.kmoe import F16, Q8_0, PagedKV

    kv = PagedKV(F16 if c["t"] == "f16" else Q8_0, c["kv"], c["hd"], c["page"])
    if c["kind"] == "copy":
        ctx.pages_copy(kv, s["pool"], s["src"], s["dst"], n_layer=c["layers"])
        return s["pool"]
    batch = ctx.paged_batch(s["table"], s["seq_len"], s["row_start"], s["s_rows"])
    if c["kind"] == "attn":
        return ctx.paged_attention(kv, s["pages"], batch, s["q"], c["heads"], window=c["window"], n_sink=c["sink"])
    n, w = c["heads"] * c["hd"], c["kv"] * c["hd"]
    x = s["qkv"]
    q = ctx.paged_rope_kv_store(kv, s["pages"], batch, x[:, :n], x[:, n:n + w], x[:, n + w:], c["heads"], c["hd"],
                                s["inv_freq"], bool(c["neox"]))
    k, v = ctx.paged_kv_read(kv, s["pages"], batch)
    return dict(q=q, k=k, v=v)


def _seen(c, n, rows):
    """Positions that the rows of a sequence of n positions see, together and at least once."""
    pairs, first = 0, n - rows
    w, k = c["window"], c["sink"]
    if not w:
        return sum(range(first + 1, n + 1)), n
    for p in range(first, n):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(k, lo)
    lo = max(0, first - w + 1)
    return pairs, n - lo + min(k, lo)


def work(case):
    c = case
    per = c["hd"] * 2 if c["t"] == "f16" else c["hd"] // 32 * 34  # one position of one kv head, K or V
    if c["kind"] == "copy":
        return dict(bytes=2 * c["n"] * c["layers"] * _page_bytes(c), flops=0)
    rows = _rows(c)
    S = sum(rows)
    if c["kind"] == "store":  # q, k, v once in; q out, k and v into the cache, out of it and out
        w = c["kv"] * c["hd"]
        return dict(bytes=S * (4 * (2 * c["heads"] * c["hd"] + 2 * w) + 2 * c["kv"] * 2 * per + 4 * w),
                    flops=S * (c["heads"] + c["kv"]) * c["hd"] * 3)
    pairs = once = 0
    for n, r in zip(_lens(c), rows):
        p, o = _seen(c, n, r)
        pairs, once = pairs + p, once + o
    return dict(bytes=once * c["kv"] * 2 * per + S * c["heads"] * c["hd"] * 8, flops=4 * pairs * c["heads"] * c["hd"])


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
    scale = s["pages"].view(torch.float16)[j // 2].double()
    return s["pages"].view(torch.int8)[o + i].double() * scale


def exact(case, seed):
    if case["kind"] == "copy":
        return None
    s = prepare(case, seed)
    c = s["case"]
    nh, kv, hd, pg = c["heads"], c["kv"], c["hd"], c["page"]
    lens = s["seq_len"].tolist()
    start = s["row_start"].tolist() if s["row_start"] is not None else list(range(len(lens) + 1))
    if c["kind"] == "store":
        S = s["s_rows"]
        pos = torch.cat([torch.arange(n - (start[b + 1] - start[b]), n, device=DEV) for b, n in enumerate(lens)])
        x = s["qkv"].double().view(S, nh + 2 * kv, hd)
        ang = (pos.to(torch.float32)[:, None] * s["inv_freq"][None, :]).double()  # rounded to 32 bits by definition
        z = torch.polar(torch.ones_like(ang), ang)[:, None, :]
        qk = x[:, :nh + kv]
        if c["neox"]:
            y = torch.view_as_real(torch.complex(qk[..., :hd // 2], qk[..., hd // 2:]) * z).transpose(-1, -2).reshape(S, nh + kv, hd)
        else:
            y = torch.view_as_real(torch.view_as_complex(qk.contiguous().view(S, nh + kv, hd // 2, 2)) * z).reshape(S, nh + kv, hd)

        def held(t):  # the values that the cache then stands for
            if c["t"] == "f16":
                return t.reshape(S, kv * hd)
            t = t.reshape(S, kv * hd // 32, 32)
            d = (t.abs().amax(-1, keepdim=True) / 127.0).half().double()
            return (torch.clamp(torch.round(t / d.clamp_min(1e-30)), -127, 127) * d).reshape(S, kv * hd)

        return dict(q=y[:, :nh].reshape(S, nh * hd), k=held(y[:, nh:]), v=held(x[:, nh + kv:]))
    out = []
    for b, n in enumerate(lens):
        r = start[b + 1] - start[b]
        p = torch.arange(n, device=DEV)
        base = s["table"][b].long()[p // pg]
        k, v = _element(s, base, p % pg, _k_at, _ks_at), _element(s, base, p % pg, _v_at, _vs_at)
        q = s["q"][start[b]:start[b + 1]].double().view(r, kv, nh // kv, hd).permute(1, 2, 0, 3)  # [kv, G, r, hd]
        o = torch.empty(kv, nh // kv, r, hd, dtype=torch.float64, device=DEV)
        for i in range(0, r, 256):  # rows at a time
            at = torch.arange(n - r + i, min(n, n - r + i + 256), device=DEV)[:, None]
            x = torch.matmul(q[:, :, i:i + 256].reshape(kv, -1, hd), k.transpose(1, 2).contiguous()).view(kv, nh // kv, -1, n) / hd ** 0.5
            hide = p[None] > at
            if c["window"]:
                hide = hide | ((at - p[None] >= c["window"]) & (p[None] >= c["sink"]))
            w = torch.softmax(x.masked_fill(hide, -math.inf), dim=-1)
            o[:, :, i:i + 256] = torch.matmul(w.reshape(kv, -1, n), v).view(kv, nh // kv, -1, hd)
        out.append(o.permute(2, 0, 1, 3).reshape(r, nh * hd))
    return torch.cat(out)
