"""A whole decode stack on one GPU: Transformer::forward
(crates/kestrel-engine/src/transformer.rs:278-302, 375-467) over libkmoe's
kernels, with every weight, the KV cache and the activations resident in HBM.

The model is given as kestrel's Transformer sees it: hyperparameters and GGUF
tensors by name (type, dims with the contiguous dimension first, bytes), so a
GGUF or KGUF reader hands its tensors over unchanged:

    hp:      arch, n_layer, n_embd, n_head, n_head_kv, head_dim, rope_dim,
             rope_freq_base, rms_eps, n_ctx, n_batch; MoE models add
             n_expert, n_expert_used, norm_topk, weights_scale
    tensors: "token_embd.weight", "output_norm.weight", optional
             "output.weight" (tied to the embedding when absent),
             "rope_freqs.weight"; per layer "blk.{l}.attn_norm.weight",
             attn_{q,k,v,output}.weight, optional attn_{q,k,v}.bias and
             attn_{q,k}_norm.weight, ffn_norm.weight, then either dense
             ffn_{gate,up,down}.weight or routed ffn_gate_inp.weight +
             ffn_{gate,up,down}_exps.weight (+ the *_shexp shared expert).

Layers with routed experts go through kmoe_moe_ffn and its HBM expert tier;
the rest through the decoder ops of include/kmoe.h. A single-token decode
step reads its position from a device counter, so it is captured once as a
HIP graph and replayed for every later token (decoding keeps the sampled
token on the device too, the largest logit's or one drawn by given random
numbers). PagedDecoder runs many sequences together over a paged key-value
cache, with the pages that they share read once or a choice of pages read at all.
"""
from __future__ import annotations

import numpy as np

from .kmoe import BLOCK, F16, F32, Q8_0, STATUS, Context, KmoeError, PagedKV, Pages, bytes_for


def _nbytes(t: int, dims) -> int:
    rows = int(np.prod(dims[1:])) if len(dims) > 1 else 1
    return bytes_for(t, dims[0]) * rows


class Decoder:
    """Transformer::forward on the GPU (see the module docstring)."""

    def __init__(self, ctx: Context, hp: dict, tensors: dict, layer_base: int = 1000):
        torch = ctx.torch
        self.ctx, self.hp, self.torch = ctx, hp, torch
        self.d, self.nh, self.nkv, self.hd = hp["n_embd"], hp["n_head"], hp["n_head_kv"], hp["head_dim"]
        self.rd, self.eps = hp["rope_dim"], float(hp["rms_eps"])
        self.neox = hp["arch"] != "llama"
        self.n_ctx, self.n_batch = hp["n_ctx"], max(1, hp.get("n_batch", 512))
        self.n_layer = hp["n_layer"]
        if self.nh % self.nkv:
            raise ValueError("n_head must be a multiple of n_head_kv")
        dev = f"cuda:{ctx.device}"
        self.dev = dev
        self._raw = {}

        def raw(name):
            ty, dims, b = tensors[name]
            b = np.ascontiguousarray(b, dtype=np.uint8).reshape(-1)
            if b.size < _nbytes(ty, dims):
                raise ValueError(f"{name}: {b.size} bytes < {_nbytes(ty, dims)}")
            t = torch.from_numpy(b).to(dev)
            self._raw[name] = (ty, list(dims), t)
            return self._raw[name]

        def vec(name):
            """An F32/F16/quantized vector as f32 on the device (dequantized by the device row kernel)."""
            ty, dims, t = raw(name)
            n = int(np.prod(dims))
            if ty == F32:
                return t[:4 * n].view(torch.float32).clone()
            return ctx.get_rows(ty, t, 1, n, [0]).reshape(n)

        self.embed = raw("token_embd.weight")
        self.n_vocab = self.embed[1][1]
        self.out_norm = vec("output_norm.weight")
        self.head = raw("output.weight") if "output.weight" in tensors else self.embed
        inv = None
        freqs = vec("rope_freqs.weight") if "rope_freqs.weight" in tensors else None
        base = np.float32(hp["rope_freq_base"])
        e = (-(2.0 * np.arange(self.rd // 2, dtype=np.float32)) / np.float32(self.rd)).astype(np.float32)
        inv = torch.from_numpy(np.power(base, e, dtype=np.float32)).to(dev)
        if freqs is not None:
            inv = inv / freqs
        self.inv_freq = inv.contiguous()

        kvw = self.nkv * self.hd
        self.layers = []
        for l in range(self.n_layer):
            p = f"blk.{l}."
            L = {"attn_norm": vec(p + "attn_norm.weight"), "ffn_norm": vec(p + "ffn_norm.weight"),
                 "wo": raw(p + "attn_output.weight")}
            wq, wk, wv = (tensors[p + f"attn_{n}.weight"] for n in "qkv")
            if wq[0] == wk[0] == wv[0]:  # one matmul over the concatenated rows (rows are independent)
                cat = np.concatenate([np.ascontiguousarray(w[2], dtype=np.uint8).reshape(-1)[:_nbytes(w[0], w[1])]
                                      for w in (wq, wk, wv)])
                L["wqkv"] = (wq[0], [wq[1][0], self.nh * self.hd + 2 * kvw], torch.from_numpy(cat).to(dev))
            else:
                L["wq"], L["wk"], L["wv"] = (raw(p + f"attn_{n}.weight") for n in "qkv")
            for n in "qkv":
                if p + f"attn_{n}.bias" in tensors:
                    L["b" + n] = vec(p + f"attn_{n}.bias")
            for n in "qk":
                if p + f"attn_{n}_norm.weight" in tensors:
                    L[n + "_norm"] = vec(p + f"attn_{n}_norm.weight")
            if p + "ffn_gate_exps.weight" in tensors:
                L["moe"] = self._moe_layer(l, layer_base + l, tensors)
            else:
                wg, wu = tensors[p + "ffn_gate.weight"], tensors[p + "ffn_up.weight"]
                if wg[0] == wu[0] and list(wg[1]) == list(wu[1]):  # gate | up rows in one matmul
                    cat = np.concatenate([np.ascontiguousarray(w[2], dtype=np.uint8).reshape(-1)[:_nbytes(w[0], w[1])]
                                          for w in (wg, wu)])
                    L["wgu"] = (wg[0], [wg[1][0], 2 * wg[1][1]], torch.from_numpy(cat).to(dev))
                else:
                    L["gate"], L["up"] = raw(p + "ffn_gate.weight"), raw(p + "ffn_up.weight")
                L["down"] = raw(p + "ffn_down.weight")
            self.layers.append(L)
        self._make_cache()
        self.cached = 0
        self.pos_dev = torch.zeros(1, dtype=torch.int32, device=dev)
        self.token_dev = torch.zeros(1, dtype=torch.int32, device=dev)
        self._graphs = {}  # by kind of step: the graph, and what it was captured for (_key)
        self._graph_bufs = None

    def _make_cache(self):
        for L in self.layers:
            for n in ("kc", "vc"):
                L[n] = self.torch.zeros((self.n_ctx, self.nkv * self.hd), dtype=self.torch.int16, device=self.dev)

    def _moe_layer(self, l: int, lid: int, tensors: dict) -> int:
        ctx, hp, p = self.ctx, self.hp, f"blk.{l}."
        E = hp["n_expert"]
        g, u, dn = (tensors[p + f"ffn_{n}_exps.weight"] for n in ("gate", "up", "down"))
        ff = g[1][1]
        ctx.layer_create(lid, E, hp["n_expert_used"], self.d, ff, g[0], u[0], dn[0], hp.get("norm_topk", True),
                         hp.get("weights_scale", 0.0))
        rty, rdims, rb = tensors[p + "ffn_gate_inp.weight"]
        if rty != F32:
            raise ValueError("the router (ffn_gate_inp) must be F32, as kestrel's moe_ffn reads it")
        ctx.router_upload(lid, np.ascontiguousarray(rb, dtype=np.uint8).view(np.float32)[:E * self.d].reshape(E, self.d))
        for k, (ty, dims, b) in enumerate((g, u, dn)):
            b = np.ascontiguousarray(b, dtype=np.uint8).reshape(-1)
            sl = _nbytes(ty, dims) // E
            for e in range(E):
                ctx.expert_upload(lid, e, k, b[e * sl:(e + 1) * sl])
        if p + "ffn_gate_shexp.weight" in tensors:
            ts = [tensors[p + f"ffn_{n}_shexp.weight"] for n in ("gate", "up", "down")]
            gi = None
            if p + "ffn_gate_inp_shexp.weight" in tensors:
                gty, gdims, gb = tensors[p + "ffn_gate_inp_shexp.weight"]
                if gty != F32:
                    raise ValueError("ffn_gate_inp_shexp must be F32")
                gi = np.ascontiguousarray(gb, dtype=np.uint8).view(np.float32)[:self.d]
            ctx.shared_expert(lid, ts[0][1][1], [t[0] for t in ts], *[t[2] for t in ts], gate_inp=gi)
        return lid

    # ------------------------------------------------------------------ steps
    def _mm(self, w, x):
        ty, dims, t = w
        return self.ctx.matmul(ty, t, int(np.prod(dims[1:])), dims[0], x)

    def _layer(self, L, x, f_prev, S: int, pos0: int, pos_dev, spare=None):
        """One decoder layer on the residual stream x [S, d]. f_prev, the
        previous layer's FFN output, joins x in the first norm's fused add.
        Returns the layer's own FFN output and the buffer that now holds the
        residual stream: x (updated in place), or spare, a second buffer that
        one-token layers write x + f_prev into (x is then left as it was)."""
        ctx, nh, nkv, hd = self.ctx, self.nh, self.nkv, self.hd
        kvw, nq = nkv * hd, nh * hd
        plain = not any(n in L for n in ("bq", "bk", "bv", "q_norm", "k_norm"))
        if "wqkv" in L and S == 1 and plain:
            # one token: the projection kernel takes the residual add and the
            # norm (into the other buffer), applies RoPE and fills the caches
            ty, dims, t = L["wqkv"]
            xr = x if spare is None else spare
            qr = ctx.norm_matmul_rope_kv(x, L["attn_norm"], self.eps, ty, t, dims[0], nh, nkv, hd, self.rd, pos0,
                                         self.inv_freq, self.neox, self.n_ctx, L["kc"], L["vc"], y=f_prev,
                                         pos_dev=pos_dev, x_out=spare)
            return self._attn_ffn(L, xr, qr, S, pos0, pos_dev), xr
        if "wqkv" in L:
            ty, dims, t = L["wqkv"]
            qkv = ctx.norm_matmul(x, L["attn_norm"], self.eps, ty, t, dims[1], dims[0], y=f_prev)
            q, k, v = qkv[:, :nq], qkv[:, nq:nq + kvw], qkv[:, nq + kvw:]
            if S > 1:
                q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        else:
            h = ctx.rmsnorm(x, L["attn_norm"], self.eps, y=f_prev)
            q, k, v = self._mm(L["wq"], h), self._mm(L["wk"], h), self._mm(L["wv"], h)
        for n, y in (("q", q), ("k", k), ("v", v)):
            if "b" + n in L:
                ctx.add_rows(y, L["b" + n])
        if "q_norm" in L:
            ctx.rmsnorm(q, L["q_norm"], self.eps, out=q)
        if "k_norm" in L:
            ctx.rmsnorm(k, L["k_norm"], self.eps, out=k)
        qr = ctx.rope_kv_store(q, k, v, nh, nkv, hd, self.rd, pos0, self.inv_freq, self.neox, self.n_ctx, L["kc"],
                               L["vc"], pos_dev)
        return self._attn_ffn(L, x, qr, S, pos0, pos_dev), x

    def _attn_ffn(self, L, x, qr, S, pos0, pos_dev):
        """Attention from the rotated q and the caches, its projection, then the FFN."""
        ctx, nh, nkv, hd = self.ctx, self.nh, self.nkv, self.hd
        ty, dims, t = L["wo"]
        o = ctx.attention_matmul(qr, L["kc"], L["vc"], nh, nkv, hd, pos0, self.n_ctx, ty, t,
                                 int(np.prod(dims[1:])), pos_dev)
        return self._ffn(L, x, o, S)

    def _ffn(self, L, x, o, S):
        """The FFN of the attention's output o added to x."""
        ctx = self.ctx
        if "moe" in L:
            # x += o, the norm of x, then the routed experts (one token: the
            # router kernel takes the norm)
            return ctx.norm_moe_ffn(L["moe"], x, L["ffn_norm"], self.eps, y=o)
        if "wgu" in L:
            ty, dims, t = L["wgu"]
            ff = dims[1] // 2
            gu = ctx.norm_matmul(x, L["ffn_norm"], self.eps, ty, t, dims[1], dims[0], y=o)
            g, u = gu[:, :ff], gu[:, ff:]
            if S > 1:
                g, u = g.contiguous(), u.contiguous()
        else:
            h = ctx.rmsnorm(x, L["ffn_norm"], self.eps, y=o)
            g, u = self._mm(L["gate"], h), self._mm(L["up"], h)
        return self._mm(L["down"], ctx.swiglu(g, u))

    def _stack(self, x, S: int, pos0: int, pos_dev):
        """All layers and the head; returns the logits of the last row."""
        f = None
        spare = self.torch.empty_like(x) if S == 1 else None  # the residual stream's second buffer
        for L in self.layers:
            f, xr = self._layer(L, x, f, S, pos0, pos_dev, spare)
            if xr is not x:
                x, spare = xr, x
        ty, dims, t = self.head
        return self.ctx.norm_matmul(x[S - 1:S], self.out_norm, self.eps, ty, t, dims[1], dims[0],
                                    y=f[S - 1:S]).reshape(-1)

    def forward(self, tokens):
        """Transformer::forward: feed host token ids; returns the last row's
        logits (f32 [n_vocab], on the device)."""
        tokens = [int(t) for t in tokens]
        if not tokens:
            raise ValueError("forward() needs at least one token")
        if self.cached + len(tokens) > self.n_ctx:
            raise ValueError(f"context full: need {self.cached + len(tokens)}, n_ctx {self.n_ctx}")
        logits = None
        for i in range(0, len(tokens), self.n_batch):
            chunk = tokens[i:i + self.n_batch]
            ty, dims, t = self.embed
            x = self.ctx.get_rows(ty, t, dims[1], dims[0], chunk)
            logits = self._stack(x, len(chunk), self.cached, None)
            self.cached += len(chunk)
        return logits

    # --------------------------------------------------------- greedy decode
    def _key(self):
        """What a captured step depends on besides its buffers: the workspaces' addresses and the regime's kernels."""
        return self.ctx.workspace_generation(), self.ctx.regime()

    def _captured(self, kind, body, rewind):
        """The graph of a step: captured anew where a workspace that it points into was reallocated since (a longer prompt
        chunk, another caller of the context), or the regime is another."""
        graph, key = self._graphs.get(kind, (None, None))
        if graph is not None and key == self._key():
            return graph
        torch = self.torch
        body()  # at the same shapes: grows every workspace first
        rewind()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(g):
                self.ctx.set_stream(torch.cuda.current_stream())  # the capturing stream
                body()
        finally:
            self.ctx.set_stream(torch.cuda.current_stream())
        self._graphs[kind] = (g, self._key())
        torch.cuda.synchronize()
        return g

    def _sampling(self, b, rows: int, u, n: int, **how):
        """The settings of a sampled decode into buffers of b, and its random numbers [n, rows] on the device."""
        torch = self.torch
        u = torch.as_tensor(u, dtype=torch.float64)
        # (below 1 stays below 1, from where on the last kept token is drawn, however little it weighs)
        u = torch.where(u < 1, u.to(torch.float32).clamp(max=1 - 2.0 ** -24), u.to(torch.float32))
        if tuple(u.shape) != (n, rows) and (rows != 1 or tuple(u.shape) != (n,)):
            raise ValueError(f"u: need [{n}, {rows}] random numbers, got {list(u.shape)}")
        vals = {}
        for name, v in how.items():
            x = np.asarray(v, dtype=np.int64 if name == "top_k" else np.float64)
            if x.shape not in ((), (rows,)):
                raise ValueError(f"{name}: one value, or one for each of {rows} sequences")
            x = np.broadcast_to(x, rows)
            vals[name] = x.clip(-1, 2 ** 31 - 1).astype(np.int32) if name == "top_k" else x.astype(np.float32)
        if "u" not in b:
            b["u"] = torch.empty(rows, dtype=torch.float32, device=self.dev)
            for name, x in vals.items():
                b[name] = torch.empty(rows, dtype=torch.int32 if name == "top_k" else torch.float32, device=self.dev)
        for name, x in vals.items():
            b[name].copy_(torch.from_numpy(x.copy()))
        return u.to(self.dev).reshape(n, rows).contiguous()

    def _decode_body(self, sampled: bool):
        b = self._graph_bufs
        ty, dims, t = self.embed
        x = self.ctx.get_rows(ty, t, dims[1], dims[0], self.token_dev, out=b["x"])
        logits = self._stack(x, 1, 0, self.pos_dev)
        b["logits"] = logits
        if sampled:
            self.ctx.sample(logits.view(1, -1), b["u"], b["temperature"], b["top_k"], b["top_p"], b["min_p"],
                            out=self.token_dev, pos_dev=self.pos_dev, advance=1)
        else:
            self.ctx.argmax(logits, out=self.token_dev, pos_dev=self.pos_dev, advance=1)

    def _decode(self, first_token: int, n: int, use_graph: bool, how):
        torch = self.torch
        if self.cached + n > self.n_ctx:
            raise ValueError("context full")
        if self._graph_bufs is None:
            self._graph_bufs = {"x": torch.empty((1, self.d), dtype=torch.float32, device=self.dev)}
        u = None if how is None else self._sampling(self._graph_bufs, 1, n=n, **how)
        self.pos_dev.fill_(self.cached)
        self.token_dev.fill_(int(first_token))
        out = torch.empty(n, dtype=torch.int32, device=self.dev)
        step = lambda: self._decode_body(u is not None)  # noqa: E731
        if use_graph:
            pos, tok = self.pos_dev.clone(), self.token_dev.clone()
            if u is not None:
                self._graph_bufs["u"].copy_(u[0] if n else torch.zeros(1))

            def rewind():
                self.pos_dev.copy_(pos)
                self.token_dev.copy_(tok)

            step = self._captured("greedy" if u is None else "sampled", step, rewind).replay
        for i in range(n):
            if u is not None:
                self._graph_bufs["u"].copy_(u[i])
            step()
            out[i:i + 1].copy_(self.token_dev)
        self.cached += n
        return out

    def decode_greedy(self, first_token: int, n: int, use_graph: bool = True):
        """Greedy decoding (sampler.rs:58-59): feed first_token, then each
        argmax, n steps; returns the n sampled ids. One step = one token
        through every layer, the head and argmax, all on the device; with
        use_graph the step is captured once and replayed."""
        return self._decode(first_token, n, use_graph, None)

    def decode_sample(self, first_token: int, n: int, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                      use_graph: bool = True):
        """decode_greedy with the tokens drawn by Context.sample: u holds n random numbers in [0, 1), the caller's; the
        settings are single numbers, read when the steps run."""
        return self._decode(first_token, n, use_graph, dict(u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))

    def close(self):
        for L in self.layers:
            if "moe" in L:
                self.ctx.layer_destroy(L["moe"])
        self.layers = []
        self._graphs = {}


class PagedDecoder(Decoder):
    """A Decoder for many sequences at once over one paged key-value cache of
    n_pages pages, F16 or Q8_0: every call takes new tokens of any of them,
    prompts and single tokens together. Sequences are numbered by the caller and
    begin with their first tokens; forks share pages until one of them writes.
    With a window a row sees the last `window` positions and the first n_sink,
    and pages that no later row sees are free again after a call, or during it
    where its new positions find no pages all at once: then each part of it
    (hp["n_batch"] rows of forward, as many greedy steps as a page has positions)
    takes its pages before it runs. head_dim 64 or 128; a sequence has at most
    hp["n_ctx"] positions, a call at most 4096 sequences, and hp["n_batch"] rows at
    a time of a forward call go through the layers.

    With share_prefixes the pages that several of a call's sequences hold in common
    (forks of a prompt) are read once for all of them (Pages.groups finds them). With
    select > 0 the attention of decode steps, and of forward calls with one token for each
    sequence, goes over that many pages for each kv head: a row's own, the first
    select_first and those whose bounds promise the largest scores; other calls go over
    all. Neither goes with a window, nor with the other."""

    # positions by kv heads and dims that would be read again (members less one, times those in common) from which a
    # group is made, with up to four heads a kv head: the 8 .. 12 us a layer that reading them once takes more (measured
    # for 32 heads over 8 of 128: 45000 positions; 16 over 4: 100000; 16 over 8 of 64, Q8_0: 110000; 32 over 4: 190000).
    # Decode steps always read such groups' pages once, as what they share is known here; prompt chunks, whose rows fill the
    # matrix tiles more or less, leave it to the call's own count of tiles.
    SHARE_LEAST = 45000 * 8 * 128

    def __init__(self, ctx: Context, hp: dict, tensors: dict, n_pages: int, page: int = 64, kv_type: int = F16,
                 window: int = 0, n_sink: int = 0, layer_base: int = 1000, share_prefixes: bool = False, select: int = 0,
                 select_first: int = 1):
        if hp["head_dim"] not in (64, 128):
            raise ValueError(f"head_dim {hp['head_dim']}: the paged cache has heads of 64 or 128")
        if kv_type not in (F16, Q8_0):
            raise ValueError("kv_type: F16 or Q8_0")
        if window < 0 or n_sink < 0 or (n_sink and not window):
            raise ValueError("window and n_sink: not negative, and n_sink with a window only")
        if page not in (32, 64, 128, 256):
            raise ValueError(f"page {page}: 32, 64, 128 or 256 positions")
        if select < 0 or (select and not 0 <= select_first < select):
            raise ValueError("select and select_first: not negative, and fewer first pages than selected ones")
        if (share_prefixes or select) and window or (share_prefixes and select):
            raise ValueError("share_prefixes, select and window: one of them at most")
        self.share_prefixes, self.select, self.select_first = share_prefixes, select, select_first
        self.account = Pages(n_pages, page)
        self.kv = PagedKV(kv_type, hp["n_head_kv"], hp["head_dim"], page)
        self.n_pages, self.window, self.n_sink = n_pages, window, n_sink
        super().__init__(ctx, hp, tensors, layer_base)
        self.cols = -(-self.n_ctx // page)
        self._graph_n = 0

    def _make_cache(self):
        self.pages = self.torch.zeros((self.n_layer, self.n_pages, self.kv.page_bytes), dtype=self.torch.uint8,
                                      device=self.dev)
        self.bounds = None
        if self.select:
            self.bounds = self.torch.zeros((self.n_layer, self.n_pages, self.nkv, 2, self.hd), dtype=self.torch.float16,
                                           device=self.dev)

    # ---------------------------------------------------------- sequences
    def length(self, seq: int) -> int:
        """Positions of seq in the cache; 0 where there is no such sequence."""
        try:
            return self.account.length(seq)
        except KmoeError:
            return 0

    def fork(self, src: int, dst: int, n: int | None = None):
        """A new sequence dst of the first n positions of src (all of them by default)."""
        self.account.fork(src, dst, self.account.length(src) if n is None else n)

    def truncate(self, seq: int, n: int):
        self.account.truncate(seq, n)

    def drop(self, seq: int):
        self.account.drop(seq)

    def compact(self, most: int | None = None) -> int:
        """Moves used pages to the front of the cache, at most `most`; how many were moved."""
        src, dst = self.account.compact(most)
        self._copy(list(zip(src.tolist(), dst.tolist())))
        if self.bounds is not None and len(src):
            s, d = (self.torch.from_numpy(x.astype(np.int64)).to(self.dev) for x in (src, dst))
            self.bounds[:, d] = self.bounds[:, s]
        return len(src)

    def _copy(self, pairs):
        if pairs:
            self.ctx.pages_copy(self.kv, self.pages, [s for s, _ in pairs], [d for _, d in pairs], self.n_layer)

    def _reserve(self, want: dict, steps=()):
        """Positions for new tokens {sequence: n}, all of them or none: the lengths before (None: a new sequence),
        and whether the call's steps {sequence: n} have to take theirs one by one, as a window's pages become free."""
        if not want or len(want) > 4096:
            raise ValueError(f"{len(want)} sequences: a call takes 1 to 4096")
        had = {}
        for s, n in want.items():
            try:
                had[s] = self.account.length(s)
            except KmoeError:
                had[s] = None
            if (had[s] or 0) + n > self.n_ctx:
                raise ValueError(f"context full: sequence {s} needs {(had[s] or 0) + n}, n_ctx {self.n_ctx}")
        try:
            copies = self.account.append_many(want)
        except KmoeError as e:
            if STATUS.get(e.status) != "BUDGET" or not self.window or len(steps) < 2:
                raise
        else:
            try:
                self._copy(copies)
            except BaseException:
                self._back(had)
                raise
            return had, False
        trial = self.account.clone()  # (fails here, or not at all)
        try:
            for step in steps:
                trial.append_many(step)
                self._trim(step, had, trial)
        finally:
            trial.close()
        return had, True

    def _append(self, want: dict):
        self._copy(self.account.append_many(want))

    def _back(self, had: dict):
        for s, n in had.items():
            if n is not None:
                self.account.truncate(s, n)
            elif self.length(s):
                self.account.drop(s)

    def _trim(self, seqs, had=None, account=None):
        """Gives up what no later row sees; with `had` not yet what the sequences need at those lengths."""
        if self.window:
            for s in seqs:
                (account or self.account).trim(s, self.window, max(self.n_sink, had[s] or 0) if had else self.n_sink)

    # -------------------------------------------------------------- steps
    def _attend(self, l: int, batch, q):
        """The batch's attention over layer l's pages, in the form that the batch asks for."""
        ctx, pages = self.ctx, self.pages[l]
        if self.select:
            ctx.paged_bounds(self.kv, pages, batch, self.bounds[l])
            if batch.steps:
                return ctx.paged_attention_selected(self.kv, pages, self.bounds[l], batch, q, self.nh, self.select,
                                                    self.select_first)
        if getattr(batch, "groups", None) is not None:
            return ctx.paged_attention_shared(self.kv, pages, batch, batch.groups, q, self.nh)
        return ctx.paged_attention(self.kv, pages, batch, q, self.nh, self.window, self.n_sink)

    def _paged_layer(self, l: int, batch, x, f_prev):
        """_layer for the rows of a batch."""
        ctx, nh, nkv, hd, S, L = self.ctx, self.nh, self.nkv, self.hd, batch.s_rows, self.layers[l]
        kvw, nq = nkv * hd, nh * hd
        if "wqkv" in L:
            ty, dims, t = L["wqkv"]
            qkv = ctx.norm_matmul(x, L["attn_norm"], self.eps, ty, t, dims[1], dims[0], y=f_prev)
            q, k, v = qkv[:, :nq], qkv[:, nq:nq + kvw], qkv[:, nq + kvw:]
            if any(n in L for n in ("bq", "bk", "bv", "q_norm", "k_norm")):
                q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        else:
            h = ctx.rmsnorm(x, L["attn_norm"], self.eps, y=f_prev)
            q, k, v = self._mm(L["wq"], h), self._mm(L["wk"], h), self._mm(L["wv"], h)
        for n, y in (("q", q), ("k", k), ("v", v)):
            if "b" + n in L:
                ctx.add_rows(y, L["b" + n])
        if "q_norm" in L:
            ctx.rmsnorm(q, L["q_norm"], self.eps, out=q)
        if "k_norm" in L:
            ctx.rmsnorm(k, L["k_norm"], self.eps, out=k)
        qr = ctx.paged_rope_kv_store(self.kv, self.pages[l], batch, q, k, v, nh, self.rd, self.inv_freq, self.neox)
        return self._ffn(L, x, self._mm(L["wo"], self._attend(l, batch, qr)), S)

    def _rows(self, x, batch):
        """All layers over the batch's rows: (x, f), whose sum is the residual stream."""
        f = None
        for l in range(self.n_layer):
            f = self._paged_layer(l, batch, x, f)
        return x, f

    def _logits(self, x, f):
        ty, dims, t = self.head
        return self.ctx.norm_matmul(x, self.out_norm, self.eps, ty, t, dims[1], dims[0], y=f)

    def _batch(self, seqs, ends, counts):
        """The batch of counts[i] rows of seqs[i] that end at its position ends[i]."""
        cols = -(-max(self.account.length(s) for s in seqs) // self.kv.page)
        table, _ = self.account.table(seqs, cols)
        starts = np.concatenate([[0], np.cumsum(counts)])
        n = len(seqs)
        d = self.torch.from_numpy(np.concatenate([ends, starts, table.reshape(-1)]).astype(np.int32)).to(self.dev)
        rs = None if max(counts) == 1 else d[n:2 * n + 1]
        return self.ctx.paged_batch(d[2 * n + 1:].view(n, cols), d[:n], rs, int(starts[-1]))

    def _groups(self, seqs, rows: int):
        """The order that puts sequences with pages in common beside each other, with where their groups begin and what
        they share; None where nothing is worth sharing (or the call's rows are too many for it)."""
        if not self.share_prefixes or len(seqs) < 2 or rows * self.nh > 1 << 21:
            return None
        order, start, shared = self.account.groups(seqs, self.SHARE_LEAST * max(4, self.nh // self.nkv) // (4 * self.nkv * self.hd))
        return (order.tolist(), start, shared) if len(shared) else None

    def _parts(self, rows: dict):
        """The rows in parts of n_batch: lists of (sequence, first token, end), a sequence at most once in each."""
        parts, part, room = [], [], self.n_batch
        for s, ts in rows.items():
            i = 0
            while i < len(ts):
                m = min(room, len(ts) - i)
                part.append((s, i, i + m))
                i, room = i + m, room - m
                if not room:
                    parts.append(part)
                    part, room = [], self.n_batch
        return parts + [part] if part else parts

    def forward(self, rows: dict):
        """Feeds rows {sequence: its next tokens}; returns the logits of each one's last token [len(rows), n_vocab],
        in the order of rows. A call that fails leaves the sequences as they were."""
        rows = {int(s): [int(t) for t in ts] for s, ts in rows.items()}
        for s, ts in rows.items():
            if not ts or min(ts) < 0 or max(ts) >= self.n_vocab:
                raise ValueError(f"sequence {s}: need at least one token, each below {self.n_vocab}")
        parts, steps = self._parts(rows), all(len(ts) == 1 for ts in rows.values())
        had, by_parts = self._reserve({s: len(ts) for s, ts in rows.items()}, [{s: j - i for s, i, j in p} for p in parts])
        try:
            logits = []
            for part in parts:
                if by_parts:
                    self._append({s: j - i for s, i, j in part})
                ty, dims, t = self.embed
                done = [s for s, _, j in part if j == len(rows[s])]
                groups = self._groups([s for s, _, _ in part], sum(j - i for _, i, j in part))
                if groups:
                    part = [part[i] for i in groups[0]]
                x = self.ctx.get_rows(ty, t, dims[1], dims[0], [tk for s, i, j in part for tk in rows[s][i:j]])
                counts = [j - i for _, i, j in part]
                batch = self._batch([p[0] for p in part], [(had[s] or 0) + j for s, _, j in part], counts)
                batch.steps = steps
                if groups:
                    start, shared = (self.torch.from_numpy(g.copy()).to(self.dev) for g in groups[1:])
                    batch.groups = self.ctx.paged_groups(start, shared, always=steps)  # (chunks: the call decides)
                x, f = self._rows(x, batch)
                end = dict(zip([p[0] for p in part], np.cumsum(counts).tolist()))
                last = [end[s] - 1 for s in done]
                if last:
                    if last != list(range(len(x))):
                        x, f = (self.ctx.get_rows(F32, y, len(y), self.d, last) for y in (x, f))
                    logits.append(self._logits(x, f))
                if by_parts:
                    self._trim([s for s, _, _ in part], had)
            logits = logits[0] if len(logits) == 1 else self.torch.cat(logits)
        except BaseException:
            self._back(had)
            raise
        self._trim(rows)
        return logits

    # ------------------------------------------------------ decode steps
    def _decode_rows(self, b, sampled: bool, shared: bool):
        ty, dims, t = self.embed
        x = self.ctx.get_rows(ty, t, dims[1], dims[0], b["tok"], out=b["x"])
        b["batch"].groups = b["groups"] if shared else None
        b["logits"] = self._logits(*self._rows(x, b["batch"]))
        if sampled:
            self.ctx.sample(b["logits"], b["u"], b["temperature"], b["top_k"], b["top_p"], b["min_p"], out=b["tok"],
                            pos_dev=b["len"], advance=1)
            return
        for i in range(len(b["logits"])):
            self.ctx.argmax(b["logits"][i], out=b["tok"][i:i + 1], pos_dev=b["len"][i:i + 1], advance=1)

    def _buffers(self, n: int):
        """The buffers of steps of n sequences, which the graphs hold."""
        b, torch = self._graph_bufs, self.torch
        if b is None or self._graph_n != n:
            i32 = dict(dtype=torch.int32, device=self.dev)
            b = {"x": torch.empty((n, self.d), dtype=torch.float32, device=self.dev), "tok": torch.empty(n, **i32),
                 "len": torch.empty(n, **i32), "table": torch.empty((n, self.cols), **i32),
                 "start": torch.empty(n // 2 + 2, **i32), "shared": torch.empty(n // 2 + 1, **i32)}
            b["batch"] = self.ctx.paged_batch(b["table"], b["len"])
            b["batch"].steps = True
            b["groups"] = self.ctx.paged_groups(b["start"], b["shared"], always=True)
            self._graph_bufs, self._graph_n, self._graphs = b, n, {}
        return b

    def _decode(self, first: dict, n: int, use_graph: bool, how):
        torch, seqs = self.torch, [int(s) for s in first]
        if n < 1:
            raise ValueError("n: at least one step")
        if any(not 0 <= int(t) < self.n_vocab for t in first.values()):
            raise ValueError(f"a token is not below {self.n_vocab}")
        page = self.kv.page
        blocks = [min(page, n - i) for i in range(0, n, page)]
        had, by_blocks = self._reserve({s: n for s in seqs}, [{s: m for s in seqs} for m in blocks])
        try:
            if by_blocks:
                self._append({s: blocks[0] for s in seqs})
            b = self._buffers(len(seqs))
            u = None if how is None else self._sampling(b, len(seqs), n=n, **how)
            groups = self._groups(seqs, len(seqs))
            order = groups[0] if groups else list(range(len(seqs)))  # of the buffers' rows, among seqs
            rows = [seqs[i] for i in order]
            at = torch.tensor([(had[s] or 0) + 1 for s in rows], dtype=torch.int32)
            tok = torch.tensor([int(first[s]) for s in rows], dtype=torch.int32)
            b["table"].copy_(torch.from_numpy(self.account.table(rows, self.cols)[0]))
            b["len"].copy_(at)
            b["tok"].copy_(tok)
            if groups:
                start, shared = (np.zeros(len(b[x]), np.int32) for x in ("start", "shared"))
                start[:], shared[:len(groups[2])] = groups[1][-1], groups[2]
                start[:len(groups[1])] = groups[1]
                b["start"].copy_(torch.from_numpy(start))
                b["shared"].copy_(torch.from_numpy(shared))
                if u is not None:
                    to = torch.tensor(order, device=self.dev)
                    u = u[:, to].contiguous()
                    for x in ("temperature", "top_k", "top_p", "min_p"):
                        b[x].copy_(b[x][to])
            out = torch.empty((n, len(seqs)), dtype=torch.int32, device=self.dev)
            step = lambda: self._decode_rows(b, u is not None, bool(groups))  # noqa: E731
            if use_graph:
                if u is not None:
                    b["u"].copy_(u[0])

                def rewind():
                    b["len"].copy_(at)
                    b["tok"].copy_(tok)

                step = self._captured(("greedy" if u is None else "sampled", bool(groups)), step, rewind).replay
            for i in range(n):
                if by_blocks and i and i % page == 0:
                    self._trim(seqs, had)
                    self._append({s: blocks[i // page] for s in seqs})
                    b["table"].copy_(torch.from_numpy(self.account.table(seqs, self.cols)[0]))
                if u is not None:
                    b["u"].copy_(u[i])
                step()
                out[i].copy_(b["tok"])
            if groups:
                out = out[:, torch.tensor(np.argsort(order), device=self.dev)]
        except BaseException:
            self._back(had)
            raise
        self._trim(seqs)
        return out

    def decode_greedy(self, first: dict, n: int, use_graph: bool = True):
        """Greedy decoding of several sequences together: feeds first {sequence: token}, then each one's argmax,
        n steps; returns the sampled ids [n, len(first)]. With use_graph a step is captured once per number of
        sequences and replayed: lengths, tokens and page tables are read on the device."""
        return self._decode({int(s): t for s, t in first.items()}, n, use_graph, None)

    def decode_sample(self, first: dict, n: int, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, use_graph: bool = True):
        """decode_greedy with the tokens drawn by Context.sample: u [n, len(first)] holds the caller's random numbers in
        [0, 1); each setting is one number, or one per sequence in the order of first. A captured step reads them on the
        device, too."""
        return self._decode({int(s): t for s, t in first.items()}, n, use_graph,
                            dict(u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))

    def close(self):
        super().close()
        self.pages = self.bounds = None
        self.account.close()


__all__ = ["Decoder", "PagedDecoder", "BLOCK"]
