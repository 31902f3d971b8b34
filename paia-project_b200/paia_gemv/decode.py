"""A minimal batch-1 decode step built around the GEMV family: the layer structure of Llama-3.1-8B / Qwen2.5-7B with
synthetic weights, every projection through this library's GEMVs, everything else on the device with torch.

One token = embedding -> L x [RMSNorm -> qkv (+ bias) with RoPE fused in its epilogue -> KV-cache write ->
grouped-query attention over the cache -> o -> residual -> RMSNorm -> gate_up -> SiLU(gate) * up -> down -> residual]
-> RMSNorm -> lm_head -> argmax. The cache holds `ctx` positions (the first ctx - 1 synthetic), and the token is decoded
at position ctx - 1, so every tensor shape is fixed and a whole token captures as one CUDA graph; tokens/s = 1 / its
device time. The reference measures decode cost per token as a sum of per-op GEMV times
(paia-bench/bench/analyze_e4.py:177-196); this measures the token itself, GEMVs and the ops between them (torch:
RMSNorm, scaled-dot-product attention, SiLU x up, residual adds).

`PagedDecodeModel` is the same step for a batch of sequences of different lengths, as a server runs it: batched GEMVs,
low-rank adapters per request, rotary positions and cache write in one pass (`serve.qkv_rope_cache`), attention over a
paged cache (`serve.paged_attention`); lengths live on the device, so one captured graph decodes token after token.
"""
import torch
import torch.nn.functional as F

from . import quant, serve

MODELS = {
    "llama31_8b": dict(hidden=4096, heads=32, kv_heads=8, head_dim=128, inter=14336, vocab=128256, layers=32,
                       qkv_bias=False, rope_theta=500000.0),
    "qwen25_7b": dict(hidden=3584, heads=28, kv_heads=4, head_dim=128, inter=18944, vocab=152064, layers=28,
                      qkv_bias=True, rope_theta=1000000.0),
}


class Projection:
    """One weight matrix [N, K] in a format, on the device, with its GEMV through the library (or, for references,
    a torch fp32 dequantise-then-matmul of the same bytes). rope = (rope_rows, head_dim, pos, theta): a fused QKV
    projection whose first rope_rows rows are q / k heads, stored pair-interleaved (quant.rope_pair_rows) and rotated
    in the GEMV's epilogue (paia_gemv_rope); its output is in the natural row order."""

    def __init__(self, lib, kind, N, K, g, bias=False, rope=None):
        self.lib, self.kind, self.N, self.K, self.rope = lib, kind, N, K, rope
        W = torch.randn(N, K, device="cuda", generator=g).mul_(0.02)
        self.s = self.z = None
        if kind == "bf16":
            self.W = W.to(torch.bfloat16)
        elif kind == "fp8":
            self.W, self.s = quant.quantize_fp8_rowwise(W)
        elif kind == "int4":
            self.W, self.s = quant.quantize_int4_g128(W)
        else:
            self.W, self.s, self.z = quant.quantize_int4_asym(W)
        del W
        self.bias = (torch.randn(N, device="cuda", generator=g) * 0.02).to(torch.bfloat16) if bias else None
        self.natural = None
        if rope is not None:
            # row-wise formats: reordering the quantised rows (and their scales / zeros / bias) is reordering W
            rows, hd = rope[0], rope[1]
            perm = lambda t: None if t is None else quant.rope_pair_rows(t, rows, hd)   # noqa: E731
            self.W, self.s, self.z, self.bias = perm(self.W), perm(self.s), perm(self.z), perm(self.bias)
            j = torch.arange(N, device="cuda")
            src = j.clone()
            jh = j[:rows] % hd
            src[:rows] = j[:rows] - jh + (jh >> 1) + (jh & 1) * (hd // 2)
            self.natural = torch.empty_like(src)
            self.natural[src] = j                                    # natural row d sits at stored row natural[d]
        table = {"bf16": lib.variants, "fp8": lib.variants_fp8, "int4": lib.variants_int4,
                 "int4_asym": lib.variants_int4_asym}[kind]
        want = {"bf16": (2, 4, 4, 0, 1), "fp8": (2, 2, 4, 0, 1)}.get(kind, (4, 2, 4, 0, 1))
        self.variant = next(v["id"] for v in table if tuple(v[k] for k in "RUWSH") == want)

    def __call__(self, x, y):
        """y = W x (+ bias) through the library's default path (bf16 in and out), rotated when rope is set."""
        L, p = self.lib, (lambda t: None if t is None else t.data_ptr())
        W, xp, yp, v = self.W.data_ptr(), x.data_ptr(), y.data_ptr(), self.variant
        if self.rope is not None:
            rows, hd, pos, theta = self.rope
            L.rope(self.kind, W, p(self.s), p(self.z), xp, p(self.bias), yp, self.N, self.K, rows, hd, pos, theta)
        elif self.kind == "bf16":
            L.bf16_bias(W, xp, p(self.bias), yp, self.N, self.K, v) if self.bias is not None else \
                L.bf16(W, xp, yp, self.N, self.K, v)
        elif self.kind == "fp8":
            L.fp8_bias(W, p(self.s), xp, p(self.bias), yp, self.N, self.K, v) if self.bias is not None else \
                L.fp8(W, p(self.s), xp, yp, self.N, self.K, v)
        elif self.kind == "int4":
            L.int4_bias(W, p(self.s), xp, p(self.bias), yp, self.N, self.K, v) if self.bias is not None else \
                L.int4(W, p(self.s), xp, yp, self.N, self.K, v)
        else:
            L.int4_asym_bias(W, p(self.s), p(self.z), xp, p(self.bias), yp, self.N, self.K, v) \
                if self.bias is not None else L.int4_asym(W, p(self.s), p(self.z), xp, yp, self.N, self.K, v)
        return y

    def rows(self, x, y):
        """y[m] = W x[m] (+ bias) for every row (bf16 [M, K] and [M, N], row-major) through paia_gemv_batched."""
        p = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        self.lib.batched(self.kind, p(self.W), p(self.s), p(self.z), x.data_ptr(), p(self.bias), y.data_ptr(),
                         x.shape[0], self.N, self.K)
        return y

    def dequantised(self):
        if self.kind == "bf16":
            return self.W.float()
        if self.kind == "fp8":
            return quant.dequant_fp8(self.W, self.s)
        if self.kind == "int4":
            return quant.dequant_int4(self.W, self.s)
        return quant.dequant_int4_asym(self.W, self.s, self.z)

    def reference(self, x, y):
        """The same projection as torch fp32 dequantise-then-matmul (rotated in fp32 when rope is set), rounded to
        bf16 once (for checks)."""
        r = self.dequantised() @ x.float()
        if self.bias is not None:
            r = r + self.bias.float()
        if self.rope is not None:
            rows, hd, pos, theta = self.rope
            r = r[self.natural]
            half = hd // 2
            inv = theta ** (-torch.arange(0, hd, 2, device=r.device, dtype=torch.float64) / hd)
            ang = pos * inv
            cos = torch.cat([ang.cos(), ang.cos()]).float()
            sin = torch.cat([ang.sin(), ang.sin()]).float()
            t = r[:rows].view(-1, hd)
            rot = torch.cat([-t[:, half:], t[:, :half]], dim=1)
            r = torch.cat([(t * cos + rot * sin).reshape(-1), r[rows:]])
        y.copy_(r.to(torch.bfloat16))
        return y

    def weight_bytes(self):
        return sum(t.numel() * t.element_size() for t in (self.W, self.s, self.z) if t is not None)


class DecodeModel:
    """Synthetic weights of a model's decode path in one format, a KV cache of `ctx` positions, and the token step.
    `dims` overrides the model's sizes (small models for tests); `layers` limits the layer count."""

    def __init__(self, lib, model, kind, ctx=1024, layers=None, seed=0, dims=None):
        cfg = dict(MODELS[model])
        cfg.update(dims or {})
        if layers is not None:
            cfg["layers"] = layers
        self.cfg, self.kind, self.ctx = cfg, kind, ctx
        H, nh, nkv, hd, I, V = (cfg[k] for k in ("hidden", "heads", "kv_heads", "head_dim", "inter", "vocab"))
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.embed = (torch.randn(V, H, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
        self.layers = []
        # RoPE (rotate-half form) of q and k at the decoded position ctx - 1, in the qkv projection's epilogue
        rope = ((nh + nkv) * hd, hd, float(ctx - 1), float(cfg["rope_theta"]))
        norm = lambda: (1.0 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16).float()   # noqa: E731
        for _ in range(cfg["layers"]):
            self.layers.append({
                "norm1": norm(),
                "norm2": norm(),
                "qkv": Projection(lib, kind, (nh + 2 * nkv) * hd, H, g, bias=cfg["qkv_bias"], rope=rope),
                "o": Projection(lib, kind, H, nh * hd, g),
                "gate_up": Projection(lib, kind, 2 * I, H, g),
                "down": Projection(lib, kind, H, I, g),
                "k": (torch.randn(nkv, ctx, hd, device="cuda", generator=g)).to(torch.bfloat16),
                "v": (torch.randn(nkv, ctx, hd, device="cuda", generator=g)).to(torch.bfloat16),
            })
        self.norm_f = norm()
        self.lm_head = Projection(lib, kind, V, H, g)
        # activations, reused every token (fixed addresses, so the token captures as a CUDA graph)
        dev = dict(device="cuda", dtype=torch.bfloat16)
        self.token = torch.zeros(1, device="cuda", dtype=torch.long)
        self.h = torch.empty(H, **dev)
        self.a = torch.empty(H, **dev)
        self.qkv = torch.empty((nh + 2 * nkv) * hd, **dev)
        self.attn = torch.empty(nh * hd, **dev)
        self.o = torch.empty(H, **dev)
        self.gu = torch.empty(2 * I, **dev)
        self.m = torch.empty(I, **dev)
        self.d = torch.empty(H, **dev)
        self.logits = torch.empty(V, **dev)

    def weight_bytes(self):
        n = self.lm_head.weight_bytes()
        for lay in self.layers:
            n += sum(lay[k].weight_bytes() for k in ("qkv", "o", "gate_up", "down"))
        return n

    @staticmethod
    def _rmsnorm(x, w, out, eps=1e-5):
        """out = bf16(x * rsqrt(mean(x^2) + eps) * w), computed in fp32 (w is kept in fp32)."""
        out.copy_(F.rms_norm(x.float(), (x.numel(),), w, eps))
        return out

    def step(self, reference=False):
        """Decode one token: reads self.token, writes self.logits and the argmax into self.token. reference=True
        runs every projection as torch fp32 dequantise-then-matmul (RoPE in fp32) instead of the library's GEMVs;
        everything else is the same code in both."""
        c = self.cfg
        nh, nkv, hd, I = c["heads"], c["kv_heads"], c["head_dim"], c["inter"]
        proj = (lambda P, x, y: P.reference(x, y)) if reference else (lambda P, x, y: P(x, y))
        self.h.copy_(self.embed.index_select(0, self.token)[0])
        pos = self.ctx - 1
        for lay in self.layers:
            self._rmsnorm(self.h, lay["norm1"], self.a)
            proj(lay["qkv"], self.a, self.qkv)                  # q and k come out rotated
            lay["k"][:, pos].copy_(self.qkv[nh * hd:(nh + nkv) * hd].view(nkv, hd))
            lay["v"][:, pos].copy_(self.qkv[(nh + nkv) * hd:].view(nkv, hd))
            att = F.scaled_dot_product_attention(self.qkv[:nh * hd].view(1, nh, 1, hd), lay["k"].unsqueeze(0),
                                                 lay["v"].unsqueeze(0), enable_gqa=True)
            self.attn.copy_(att.reshape(-1))
            proj(lay["o"], self.attn, self.o)
            self.h.add_(self.o)                                  # bf16 add: fp32 sum rounded once
            self._rmsnorm(self.h, lay["norm2"], self.a)
            proj(lay["gate_up"], self.a, self.gu)
            torch.mul(F.silu(self.gu[:I]), self.gu[I:], out=self.m)
            proj(lay["down"], self.m, self.d)
            self.h.add_(self.d)
        self._rmsnorm(self.h, self.norm_f, self.a)
        proj(self.lm_head, self.a, self.logits)
        self.token.copy_(torch.argmax(self.logits).view(1))
        return self.logits


class PagedDecodeModel:
    """Synthetic weights of a model's decode path in one format and a paged KV cache for `batch` sequences of up to
    `max_len` positions (bf16, or float8_e4m3fn with a scale per kv head where cache="fp8"), the first lens[b] of them
    synthetic. step() decodes one token of every sequence at position lens[b], appends it and raises lens[b].
    adapters > 0: that many low-rank adapters of rank `rank` on the qkv, o, gate_up and down projections; self.adapter[b]
    (int32, -1: none) names the one of sequence b. qk_norm: RMS norm of q and k per head before the rotation. A sequence
    that is full must be retired by its caller; active[b] = False (self.active) makes row b padding: its cache and length
    stay, its logits are those of an empty context."""

    def __init__(self, lib, model, kind, lens, max_len=1024, page_size=16, cache="bf16", adapters=0, rank=16,
                 qk_norm=False, layers=None, seed=0, dims=None):
        cfg = dict(MODELS[model])
        cfg.update(dims or {})
        if layers is not None:
            cfg["layers"] = layers
        if not lens or max(lens) >= max_len or min(lens) < 0:
            raise ValueError(f"lens must lie in [0, max_len = {max_len}), got {lens}")
        self.lib, self.cfg, self.kind, self.page_size, self.max_len = lib, cfg, kind, page_size, max_len
        H, nh, nkv, hd, I, V = (cfg[k] for k in ("hidden", "heads", "kv_heads", "head_dim", "inter", "vocab"))
        self.batch = B = len(lens)
        g = torch.Generator(device="cuda").manual_seed(seed)
        dev = dict(device="cuda", dtype=torch.bfloat16)
        self.embed = (torch.randn(V, H, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
        norm = lambda n: (1.0 + 0.1 * torch.randn(n, device="cuda", generator=g)).to(torch.bfloat16).float()   # noqa: E731
        sizes = {"qkv": ((nh + 2 * nkv) * hd, H), "o": (H, nh * hd), "gate_up": (2 * I, H), "down": (H, I)}
        per_seq = -(-max_len // page_size)
        order = torch.randperm(B * per_seq, device="cuda", generator=g)
        self.page_table = order.view(B, per_seq).to(torch.int32)
        dtype = torch.bfloat16 if cache == "bf16" else torch.float8_e4m3fn
        self.k_scale = self.v_scale = None
        if cache != "bf16":
            self.k_scale = torch.full((nkv,), 1 / 32, device="cuda")
            self.v_scale = torch.full((nkv,), 1 / 32, device="cuda")
        self.layers = []
        for _ in range(cfg["layers"]):
            lay = {"norm1": norm(H), "norm2": norm(H), "q_norm": norm(hd) if qk_norm else None,
                   "k_norm": norm(hd) if qk_norm else None}
            for name, (n, k) in sizes.items():
                lay[name] = Projection(lib, kind, n, k, g, bias=name == "qkv" and cfg["qkv_bias"])
                if adapters:
                    lay[name + "_a"] = (torch.randn(adapters, rank, k, device="cuda", generator=g) / k ** 0.5).to(torch.bfloat16)
                    lay[name + "_b"] = (torch.randn(adapters, n, rank, device="cuda", generator=g) * 0.02).to(torch.bfloat16)
            for name in ("k", "v"):
                x = torch.randn(B * per_seq, page_size, nkv, hd, device="cuda", generator=g)
                lay[name] = (x if cache == "bf16" else x * 32).to(dtype)
            self.layers.append(lay)
        self.norm_f = norm(H)
        self.lm_head = Projection(lib, kind, V, H, g)
        self.scaling = torch.ones(adapters, device="cuda") if adapters else None
        self.adapter = torch.full((B,), -1, dtype=torch.int32, device="cuda") if adapters else None
        self.inv_freq = serve.rope_inv_freq(hd, cfg["rope_theta"])
        self.workspace = serve.attention_workspace(lib, nh, nkv, hd)
        # state and activations, at fixed addresses so that the step captures as a CUDA graph
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.active = torch.ones(B, dtype=torch.bool, device="cuda")
        self.token = torch.zeros(B, device="cuda", dtype=torch.long)
        self.positions = torch.empty(B, dtype=torch.int32, device="cuda")
        self.padding = torch.full((B,), -1, dtype=torch.int32, device="cuda")
        self.seen = torch.empty(B, dtype=torch.int32, device="cuda")
        buf = lambda n: torch.zeros(B, n, **dev)   # noqa: E731
        self.h, self.a, self.o, self.d = (buf(H) for _ in range(4))
        self.qkv, self.gu, self.m, self.logits = buf((nh + 2 * nkv) * hd), buf(2 * I), buf(I), buf(V)
        self.q, self.attn = torch.zeros(B, nh, hd, **dev), torch.zeros(B, nh, hd, **dev)

    def _project(self, lay, name, x, y):
        """y = the projection of every row, plus the row's adapter."""
        lay[name].rows(x, y)
        if self.adapter is not None:
            serve.lora(self.lib, x, lay[name + "_a"], lay[name + "_b"], self.adapter, y, base=y, scaling=self.scaling)

    def _rmsnorm(self, w, eps=1e-5):
        self.a.copy_(F.rms_norm(self.h.float(), (self.h.shape[1],), w, eps))

    def step(self):
        """One token of every active sequence: reads self.token, writes self.logits and the argmax of each active row
        into self.token, appends to the cache and raises the lengths."""
        I = self.cfg["inter"]
        self.h.copy_(self.embed.index_select(0, self.token))
        torch.where(self.active, self.lens, self.padding, out=self.positions)      # padding rows: position -1, length 0
        torch.add(self.positions, 1, out=self.seen)
        for lay in self.layers:
            self._rmsnorm(lay["norm1"])
            self._project(lay, "qkv", self.a, self.qkv)
            serve.qkv_rope_cache(self.lib, self.qkv, self.positions, self.inv_freq, self.q, lay["k"], lay["v"],
                                 self.page_table, q_norm=lay["q_norm"], k_norm=lay["k_norm"], k_scale=self.k_scale,
                                 v_scale=self.v_scale)
            serve.paged_attention(self.lib, self.q, lay["k"], lay["v"], self.page_table, self.seen, self.attn,
                                  self.workspace, k_scale=self.k_scale, v_scale=self.v_scale)
            self._project(lay, "o", self.attn.view(self.batch, -1), self.o)
            self.h.add_(self.o)
            self._rmsnorm(lay["norm2"])
            self._project(lay, "gate_up", self.a, self.gu)
            torch.mul(F.silu(self.gu[:, :I]), self.gu[:, I:], out=self.m)
            self._project(lay, "down", self.m, self.d)
            self.h.add_(self.d)
        self._rmsnorm(self.norm_f)
        self.lm_head.rows(self.a, self.logits)
        self.token.copy_(torch.where(self.active, torch.argmax(self.logits, 1), self.token))
        self.lens.add_(self.active)
        return self.logits


def time_tokens(model, tokens=20, warmup=3):
    """(device microseconds per token, the token ids decoded): the token step captured as one CUDA graph, replayed
    `tokens` times (each replay decodes the next token from the previous one's argmax)."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(warmup):
            model.step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        model.step()
    for _ in range(warmup):
        g.replay()
    torch.cuda.synchronize()
    ids = []
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(tokens):
        g.replay()
    e1.record()
    torch.cuda.synchronize()
    ids.append(int(model.token[0].item()))
    us = e0.elapsed_time(e1) * 1e3 / tokens
    del g
    return us, ids
