"""The operators of a batched decode step that sit beside the GEMVs, as cases for measurement: attention of one new
token per sequence over a paged key-value cache ("attn"), per-head norm + rotary positions + cache write of a fused
QKV projection ("rope"), and the low-rank adapters of many requests beside a shared projection ("lora").

`run` computes a case with elementary torch operations in 32 bits (64 for the rotation's angles), or, where `own` is
set, through the framework's entry points (paia_gemv.serve). `exact` is the operators' definition in 64 bits.
Lengths, ranks and row assignments follow from the case, the values and their order from the seed.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
DEV = "cuda"

# ------------------------------------------------------------------ cases

_LLAMA = dict(heads=32, kv_heads=8, head_dim=128)      # Llama-3.1-8B's attention
_QWEN = dict(heads=28, kv_heads=4, head_dim=128)       # Qwen2.5-7B's attention: 7 query heads per kv head


def listed():
    return [
        # one chat request at the decode loop's own context: latency counts
        dict(name="attn one 1k", op="attn", batch=1, **_LLAMA, page=16, cache="bf16", hnd=False, longest=1024,
             ragged=False, window=0, lse=False),
        # a server's ordinary batch: every length from a few tokens to 4k, some slots of the batch empty
        dict(name="attn ragged 32", op="attn", batch=32, **_QWEN, page=16, cache="bf16", hnd=False, longest=4100,
             ragged=True, window=0, lse=True),
        # one very long document, odd length
        dict(name="attn one 128k", op="attn", batch=1, **_LLAMA, page=16, cache="bf16", hnd=True, longest=131071,
             ragged=False, window=0, lse=False),
        # a full server: 64 requests of 8k in an FP8 cache
        dict(name="attn fp8 64x8k", op="attn", batch=64, **_LLAMA, page=64, cache="e4m3", hnd=True, longest=8190,
             ragged=False, window=0, lse=False),
        # sliding-window layers of a small model: heads of 64, no shared kv heads, the window inside a long cache
        dict(name="attn window 16", op="attn", batch=16, heads=16, kv_heads=16, head_dim=64, page=32, cache="bf16",
             hnd=False, longest=6000, ragged=True, window=1024, lse=False),
        # the decode step of one request
        dict(name="rope one token", op="rope", tokens=1, **_LLAMA, rot=128, norm=False, interleaved=False,
             cache="bf16", page=16, start=1023, run=1),
        # the decode step of a large batch with per-head norms and an FP8 cache; some rows are padding
        dict(name="rope batch fp8", op="rope", tokens=250, **_QWEN, rot=128, norm=True, interleaved=False,
             cache="e4m3", page=16, start=30000, run=1),
        # a chunk of prompts: 8 runs of tokens, far positions, norms
        dict(name="rope prompt 8k", op="rope", tokens=8192, **_LLAMA, rot=128, norm=True, interleaved=False,
             cache="bf16", page=16, start=100000, run=1024),
        # eight requests, each its own small adapter, beside the fused QKV projection
        dict(name="lora 8 qkv", op="lora", rows=8, k=4096, n=6144, rank=16, used=8, bank=16, mixed=False),
        # a server's batch: 24 adapters of mixed ranks among 61 requests, some without one, beside gate_up
        dict(name="lora 61 gate_up", op="lora", rows=61, k=4096, n=28672, rank=32, used=24, bank=32, mixed=True),
        # as many adapters as requests at rank 64, beside down
        dict(name="lora 128 down", op="lora", rows=128, k=14336, n=4096, rank=64, used=128, bank=128, mixed=False),
        # a prompt of one tenant: every row the same adapter
        dict(name="lora one 512", op="lora", rows=512, k=3584, n=4608, rank=64, used=1, bank=4, mixed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rope", "lora"])
    if op == "attn":
        kv = rng.choice([1, 2, 4, 8])
        hd = rng.choice([64, 96, 128, 128, 256])
        heads = kv * rng.choice([1, 2, 4, 5, 7, 8, 16])
        batch = _log(rng, 1, 128)
        longest = _log(rng, 1, 131072)
        cache = rng.choice(["bf16", "e4m3"])
        while batch * longest * kv * hd > 64 * 8190 * 8 * 128 / 2:
            longest = (longest + 1) // 2
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv, head_dim=hd, page=rng.choice([8, 16, 32, 64, 128]),
                    cache=cache, hnd=rng.random() < 0.5, longest=longest, ragged=rng.random() < 0.6,
                    window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0, lse=rng.random() < 0.3)
    if op == "rope":
        kv = rng.choice([1, 2, 4, 8])
        hd = rng.choice([64, 96, 128, 128, 256])
        heads = kv * rng.choice([1, 2, 4, 7])
        tokens = _log(rng, 1, 8192)
        while tokens * (heads + 2 * kv) * hd > 8192 * 48 * 128:
            tokens = (tokens + 1) // 2
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, head_dim=hd,
                    rot=rng.choice([hd, hd, hd // 2]), norm=rng.random() < 0.7, interleaved=rng.random() < 0.3,
                    cache=rng.choice(["bf16", "bf16", "e4m3"]), page=rng.choice([8, 16, 32, 64]),
                    start=_log(rng, 1, 120000), run=rng.choice([1, 1, 7, 64, 500]))
    k = 8 * _log(rng, 64, 1792)
    n = 8 * _log(rng, 64, 3584)
    rank = rng.choice([8, 16, 32, 64])
    rows = _log(rng, 1, 512)
    while rows * rank * (k + n) > 128 * 64 * (14336 + 4096):
        rows = (rows + 1) // 2
    used = max(1, min(rows, _log(rng, 1, 128)))
    return dict(op=op, rows=rows, k=k, n=n, rank=rank, used=used, bank=used + rng.randrange(0, 9),
                mixed=rng.random() < 0.5)


# ------------------------------------------------------------------ what a case holds

def _lengths(case):
    """Sequence lengths of an attention case: all `longest`, or spread from a few tokens to `longest` (more short ones
    than long), with empty slots."""
    b, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * b
    spread = [max(1, round(longest * ((i * 0.6180339887 + 0.37) % 1.0) ** 2)) for i in range(b)]
    return [longest if i == 0 else 0 if i % 13 == 7 else v for i, v in enumerate(spread)]


def _rope_rows(case):
    """(sequence, position) of each row of a rope case: runs of `run` consecutive tokens, each run another sequence;
    where there are more than 15 sequences of one token, one row in 16 is padding (position -1)."""
    rows, t, s = [], 0, 0
    while t < case["tokens"]:
        first = case["start"] + 37 * s
        n = min(case["run"], case["tokens"] - t)
        rows += [(s, -1 if case["run"] == 1 and s % 16 == 15 else first + i) for i in range(n)]
        t, s = t + n, s + 1
    return rows


def _lora_rows(case):
    """(slot of each row (-1: no adapter), rank of each slot)."""
    slots = [-1 if case["mixed"] and m % 5 == 4 else m % case["used"] for m in range(case["rows"])]
    ranks = [max(8, case["rank"] >> (a % 3)) if case["mixed"] else case["rank"] for a in range(case["used"])]
    return slots, ranks


def work(case):
    if case["op"] == "attn":
        w = case["window"]
        tokens = sum(min(v, w) if w else v for v in _lengths(case))
        es = 2 if case["cache"] == "bf16" else 1
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        return {"bytes": 2 * tokens * kv * hd * es + 4 * case["batch"] * h * hd, "flops": 4 * tokens * h * hd}
    if case["op"] == "rope":
        live = sum(p >= 0 for _, p in _rope_rows(case))
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        es = 2 if case["cache"] == "bf16" else 1
        return {"bytes": live * hd * (2 * (h + 2 * kv) + 2 * h + 2 * kv * es), "flops": live * (h + kv) * hd * 7}
    slots, ranks = _lora_rows(case)
    k, n, m = case["k"], case["n"], case["rows"]
    seen = {s for s in slots if s >= 0}
    return {"bytes": sum(2 * ranks[s] * (k + n) for s in seen) + 2 * m * k + 4 * m * n,
            "flops": sum(2 * ranks[s] * (k + n) for s in slots if s >= 0)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    st = dict(case=case)
    if case["op"] == "attn":
        b, hq, kv, hd, page = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim", "page"))
        lens = _lengths(case)
        lens = [lens[i] for i in torch.randperm(b, generator=h).tolist()]
        need = [-(-v // page) for v in lens]
        pages = sum(need) + 3                                    # the pool holds pages of nobody too
        order = torch.randperm(pages, generator=h).to(torch.int32)
        table = torch.full((b, max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for i, c in enumerate(need):
            table[i, :c] = order[at:at + c]
            at += c
        shape = (pages, kv, page, hd) if case["hnd"] else (pages, page, kv, hd)

        def pool():
            t = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
            t.normal_(generator=g)
            if case["cache"] == "e4m3":
                t = t.mul_(40.0).to(E4M3)                        # stored as value / scale, scales near 1 / 40
            return t.transpose(1, 2) if case["hnd"] else t       # [pages, page, kv_heads, head_dim]

        st.update(q=normal(b, hq, hd).to(torch.bfloat16), k=pool(), v=pool(), table=table.to(DEV), lens=i32(lens),
                  out=torch.zeros(b, hq, hd, dtype=torch.bfloat16, device=DEV),
                  lse=torch.zeros(b, hq, device=DEV) if case["lse"] else None, ks=None, vs=None)
        if case["cache"] == "e4m3":
            st.update(ks=(1 + 0.2 * normal(kv).clamp(-2, 2)) / 40, vs=(1 + 0.2 * normal(kv).clamp(-2, 2)) / 40)
    elif case["op"] == "rope":
        t, hq, kv, hd, page = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "page"))
        rows = _rope_rows(case)
        seqs = 1 + max(s for s, _ in rows)
        used = sorted({(s, p // page) for s, p in rows if p >= 0})
        order = torch.randperm(len(used) + 2, generator=h).tolist()
        table = torch.full((seqs, 1 + max(c for _, c in used)), -1, dtype=torch.int32)
        at = torch.tensor(used)
        table[at[:, 0], at[:, 1]] = torch.tensor(order[:len(used)], dtype=torch.int32)
        dt = torch.bfloat16 if case["cache"] == "bf16" else E4M3
        half = case["rot"] // 2
        st.update(qkv=normal(t, (hq + 2 * kv) * hd).to(torch.bfloat16), pos=i32([p for _, p in rows]),
                  seq=i32([s for s, _ in rows]), table=table.to(DEV),
                  freq=500000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half),
                  qn=1 + 0.1 * normal(hd) if case["norm"] else None, kn=1 + 0.1 * normal(hd) if case["norm"] else None,
                  q_out=torch.zeros(t, hq, hd, dtype=torch.bfloat16, device=DEV),
                  k=torch.zeros(len(order), page, kv, hd, dtype=dt, device=DEV),
                  v=torch.zeros(len(order), page, kv, hd, dtype=dt, device=DEV), ks=None, vs=None)
        if case["cache"] == "e4m3":
            st.update(ks=(1 + 0.2 * normal(kv).clamp(-2, 2)) / 40, vs=(1 + 0.2 * normal(kv).clamp(-2, 2)) / 40)
    else:
        m, k, n, r, bank = (case[x] for x in ("rows", "k", "n", "rank", "bank"))
        slots, ranks = _lora_rows(case)
        ident = torch.randperm(bank, generator=h)[:case["used"]].tolist()
        slots = [slots[i] for i in torch.randperm(m, generator=h).tolist()]
        rank_of = [r] * bank
        for s, a in enumerate(ident):
            rank_of[a] = ranks[s]
        st.update(x=normal(m, k).to(torch.bfloat16), base=normal(m, n).to(torch.bfloat16),
                  a=(normal(bank, r, k) / math.sqrt(k)).to(torch.bfloat16),
                  b=(normal(bank, n, r) * 0.02).to(torch.bfloat16),
                  adapter=i32([-1 if s < 0 else ident[s] for s in slots]), ranks=i32(rank_of),
                  scaling=2.0 + 0.1 * normal(bank), out=torch.empty(m, n, dtype=torch.bfloat16, device=DEV))
    return st


# ------------------------------------------------------------------ the framework's calls

_kept = {}                    # what a program keeps for its lifetime: the library's handle, one workspace per head layout


def _library():
    if "lib" not in _kept:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paia-project_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from paia_gemv import load_lib, serve
        _kept.update(lib=load_lib(), serve=serve)
    return _kept["lib"], _kept["serve"]


def _run_own(st):
    lib, serve = _library()
    c = st["case"]
    if c["op"] == "attn":
        key = (c["heads"], c["kv_heads"], c["head_dim"])
        ws = _kept.get(key)
        if ws is None:
            ws = _kept[key] = serve.attention_workspace(lib, *key)
        serve.paged_attention(lib, st["q"], st["k"], st["v"], st["table"], st["lens"], st["out"], ws,
                              window=c["window"], k_scale=st["ks"], v_scale=st["vs"], lse=st["lse"])
        return (st["out"], st["lse"]) if c["lse"] else st["out"]
    if c["op"] == "rope":
        serve.qkv_rope_cache(lib, st["qkv"], st["pos"], st["freq"], st["q_out"], st["k"], st["v"], st["table"],
                             seq=st["seq"], q_norm=st["qn"], k_norm=st["kn"], eps=1e-6,
                             interleaved=c["interleaved"], k_scale=st["ks"], v_scale=st["vs"])
        return st["q_out"], st["k"], st["v"]
    serve.lora(lib, st["x"], st["a"], st["b"], st["adapter"], st["out"], base=st["base"], scaling=st["scaling"],
               ranks=st["ranks"])
    return st["out"]


# ------------------------------------------------------------------ the plain forms

def _pages(pool, table):
    """fp32 [batch, positions, kv_heads, head_dim] of a paged pool (absent pages read page 0)."""
    t = table.clamp(min=0).long()
    x = pool.view(torch.uint8)[t].view(E4M3).float() if pool.dtype == E4M3 else pool[t].float()
    return x.flatten(1, 2)


def _plain_attn(st):
    c = st["case"]
    kv, group, hd = c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"]
    k, v = _pages(st["k"], st["table"]), _pages(st["v"], st["table"])
    b, length = k.shape[:2]
    q = st["q"].float().view(b, kv, group, hd) / math.sqrt(hd)
    if st["ks"] is not None:
        q = q * st["ks"].view(1, kv, 1, 1)
    s = q @ k.permute(0, 2, 3, 1)                                # [batch, kv_heads, group, positions]
    at, lens = torch.arange(length, device=DEV), st["lens"].view(b, 1)
    dead = at >= lens
    if c["window"]:
        dead = dead | (at < lens - c["window"])
    s = s.masked_fill(dead.view(b, 1, 1, length), -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill(dead.view(b, length, 1, 1), 0.0)
    o = (p @ v.permute(0, 2, 1, 3)) / total.clamp(min=1e-30)
    if st["vs"] is not None:
        o = o * st["vs"].view(1, kv, 1, 1)
    st["out"].copy_(o.view(b, -1, hd))
    if not c["lse"]:
        return st["out"]
    st["lse"].copy_((top + torch.log(total)).view(b, -1))
    return st["out"], st["lse"]


def _plain_rope(st):
    c = st["case"]
    hq, kv, hd, rot, page = (c[x] for x in ("heads", "kv_heads", "head_dim", "rot", "page"))
    live = (st["pos"] >= 0).nonzero()[:, 0]
    pos, seq = st["pos"][live].long(), st["seq"][live].long()
    x = st["qkv"][live].float().view(len(live), hq + 2 * kv, hd)
    q, k, v = x[:, :hq], x[:, hq:hq + kv], x[:, hq + kv:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * st["qn"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * st["kn"]
    angle = pos.double()[:, None] * st["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(t):
        r, rest = t[..., :rot], t[..., rot:]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)

    q, k = turn(q), turn(k)
    st["q_out"][live] = q.to(torch.bfloat16)
    where = st["table"][seq, pos // page].long(), pos % page
    if c["cache"] == "bf16":
        st["k"][where] = k.to(torch.bfloat16)
        st["v"][where] = v.to(torch.bfloat16)
    else:
        st["k"].view(torch.uint8)[where] = (k / st["ks"][:, None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
        st["v"].view(torch.uint8)[where] = (v / st["vs"][:, None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
    return st["q_out"], st["k"], st["v"]


def _plain_lora(st):
    c = st["case"]
    ad = st["adapter"].long()
    has, ad = ad >= 0, ad.clamp(min=0)
    t = (st["a"][ad].float() @ st["x"].float()[:, :, None])[..., 0]
    t = t * (torch.arange(c["rank"], device=DEV) < st["ranks"][ad][:, None])
    d = (st["b"][ad].float() @ (t * st["scaling"][ad][:, None])[:, :, None])[..., 0]
    st["out"].copy_(st["base"].float() + d * has[:, None])
    return st["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "rope": _plain_rope, "lora": _plain_lora}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits

def _to_e4m3(x):
    """The nearest e4m3 value (ties to even, at most 448), in 64 bits."""
    a = x.abs().clamp(max=448.0)
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (e - 4).clamp(min=-9))
    return torch.sign(x) * torch.round(a / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    f = torch.float64
    if case["op"] == "attn":
        kv, hd, page = case["kv_heads"], case["head_dim"], case["page"]
        out = torch.zeros(case["batch"], case["heads"], hd, dtype=f, device=DEV)
        lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=f, device=DEV)
        for b, length in enumerate(st["lens"].tolist()):
            first = max(0, length - case["window"]) if case["window"] else 0
            if length == 0:
                continue
            ids = st["table"][b, first // page:-(-length // page)].long()
            lo = first - first // page * page

            def rows(pool, scale):
                t = pool.view(torch.uint8)[ids].view(E4M3) if pool.dtype == E4M3 else pool[ids]
                t = t.flatten(0, 1)[lo:lo + length - first].to(f)
                return t if scale is None else t * scale.to(f)[:, None]

            kk, vv = rows(st["k"], st["ks"]), rows(st["v"], st["vs"])
            for j in range(kv):
                heads = slice(j * (case["heads"] // kv), (j + 1) * (case["heads"] // kv))
                s = (st["q"][b, heads].to(f) @ kk[:, j].T) * hd ** -0.5
                lse[b, heads] = torch.logsumexp(s, -1)
                out[b, heads] = torch.softmax(s, -1) @ vv[:, j]
        return (out, lse) if case["lse"] else out
    if case["op"] == "rope":
        hq, kv, hd, rot, page = (case[x] for x in ("heads", "kv_heads", "head_dim", "rot", "page"))
        x = st["qkv"].to(f).view(case["tokens"], hq + 2 * kv, hd)
        if case["norm"]:
            w = torch.ones(hq + 2 * kv, hd, dtype=f, device=DEV)
            w[:hq], w[hq:hq + kv] = st["qn"].to(f), st["kn"].to(f)
            unit = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            unit[:, hq + kv:] = x[:, hq + kv:]
            x = unit * w
        i = torch.arange(rot // 2, device=DEV)
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
        z = torch.polar(torch.ones(1, dtype=f, device=DEV), st["pos"].to(f)[:, None] * st["freq"])[:, None]
        w = torch.complex(x[:, :hq + kv, first], x[:, :hq + kv, second]) * z
        y = x.clone()
        y[:, :hq + kv, first], y[:, :hq + kv, second] = w.real, w.imag
        q = torch.where(st["pos"].view(-1, 1, 1) >= 0, y[:, :hq], 0.0)
        pools = [torch.zeros(st["k"].shape, dtype=f, device=DEV) for _ in range(2)]
        ok = st["pos"] >= 0
        p, s = st["pos"][ok].long(), st["seq"][ok].long()
        at = st["table"][s, p // page].long() * page + p % page
        for pool, rows, scale in zip(pools, (y[ok, hq:hq + kv], y[ok, hq + kv:]), (st["ks"], st["vs"])):
            if scale is not None:
                rows = _to_e4m3(rows / scale.to(f)[:, None])
            pool.view(-1, kv, hd).index_copy_(0, at, rows)
        return q, pools[0], pools[1]
    out = st["base"].to(f)
    for a in sorted(set(st["adapter"].tolist()) - {-1}):
        rows = (st["adapter"] == a).nonzero()[:, 0]
        r = int(st["ranks"][a])
        t = st["x"][rows].to(f) @ st["a"][a, :r].to(f).T
        out[rows] += float(st["scaling"][a]) * (t @ st["b"][a, :, :r].to(f).T)
    return out
