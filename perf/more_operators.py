"""The operators of a feed-forward block with experts, as cases for measurement: choosing each token's experts and grouping
the tokens by expert ("route"), the products of each group with its expert's weights ("experts"), and the norms before and
after a block with its weighted sum, gate and residual ("norm").

`run` computes a case with elementary torch operations in 32 bits (64 for the scores by which experts are chosen under
sigmoid), or, where `own` is set, through the framework's entry points (paia_gemv.serve). `exact` is the operators'
definition in 64 bits. How many tokens each expert gets follows from the case; values, tokens and their order from the seed.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
DEV = "cuda"

# ------------------------------------------------------------------ cases


def listed():
    return [
        # the decode step of one request: latency counts
        dict(name="route one token", op="route", tokens=1, experts=64, top_k=8, scoring="softmax", bias=False, renorm=True,
             logits="bf16", padded=False),
        # a server's batch, sigmoid scores with a bias that balances the experts; some rows are padding
        dict(name="route batch sigmoid", op="route", tokens=250, experts=256, top_k=8, scoring="sigmoid", bias=True,
             renorm=True, logits="f32", padded=True),
        # a chunk of prompts
        dict(name="route prompt 8k", op="route", tokens=8192, experts=128, top_k=8, scoring="softmax", bias=False,
             renorm=False, logits="bf16", padded=False),
        # one request: each of its experts has one row
        dict(name="experts one token", op="experts", tokens=1, experts=64, top_k=8, n=2048, k=4096, kind="bf16", act=True,
             gather=True, skew=0.0),
        # a server's batch over FP8 weights, some experts popular and some without a row
        dict(name="experts batch fp8", op="experts", tokens=32, experts=64, top_k=8, n=2048, k=3584, kind="fp8", act=True,
             gather=True, skew=0.7),
        # the way back down of an odd batch
        dict(name="experts down fp8 61", op="experts", tokens=61, experts=64, top_k=8, n=4096, k=1024, kind="fp8", act=False,
             gather=False, skew=0.5),
        # a chunk of prompts over few large experts: the tensor cores count
        dict(name="experts down prompt", op="experts", tokens=4096, experts=8, top_k=2, n=4096, k=14336, kind="bf16",
             act=False, gather=False, skew=0.3),
        # a chunk of prompts over many small experts in FP8
        dict(name="experts prompt fp8", op="experts", tokens=2048, experts=64, top_k=8, n=2048, k=4096, kind="fp8", act=True,
             gather=True, skew=0.5),
        # residual and norm of one request's step
        dict(name="norm one token", op="norm", tokens=1, hidden=4096, top_k=0, post=False, gate="none", pre=True, scale=1.0),
        # the end of a block with experts for a batch: weighted sum, norm after, gate, residual, norm before the next
        dict(name="norm experts 61", op="norm", tokens=61, hidden=4096, top_k=8, post=True, gate="channel", pre=True,
             scale=1.0),
        # a chunk of prompts
        dict(name="norm prompt 8k", op="norm", tokens=8192, hidden=3584, top_k=0, post=True, gate="token", pre=True,
             scale=0.5),
        dict(name="norm experts prompt", op="norm", tokens=4096, hidden=4096, top_k=2, post=False, gate="none", pre=True,
             scale=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "experts", "norm"])
    experts = rng.choice([4, 8, 16, 32, 60, 64, 100, 128, 256])
    top_k = min(experts, rng.choice([1, 2, 4, 6, 8, 8]))
    if op == "route":
        scoring = rng.choice(["softmax", "softmax", "sigmoid"])
        return dict(op=op, tokens=_log(rng, 1, 8192), experts=experts, top_k=top_k, scoring=scoring,
                    bias=scoring == "sigmoid" and rng.random() < 0.7, renorm=rng.random() < 0.6,
                    logits=rng.choice(["bf16", "f32"]), padded=rng.random() < 0.3)
    if op == "norm":
        tokens, hidden = _log(rng, 1, 8192), 8 * _log(rng, 64, 1792)
        many = rng.choice([0, 0, 1, 2, 4, 8])
        while tokens * hidden * (4 + max(0, many - 1)) > 8192 * 3584 * 4:
            tokens = (tokens + 1) // 2
        return dict(op=op, tokens=tokens, hidden=hidden, top_k=many, post=rng.random() < 0.5,
                    gate=rng.choice(["none", "channel", "token", "full"]), pre=rng.random() < 0.8,
                    scale=rng.choice([1.0, 1.0, 0.5, 0.22]))
    kind, act = rng.choice(["bf16", "fp8"]), rng.random() < 0.5
    n, k = 16 * _log(rng, 16, 512), 16 * _log(rng, 16, 896)
    while experts * n * k > 64 * 2048 * 4096:
        n, k = 16 * ((n // 16 + 1) // 2), 16 * ((k // 16 + 1) // 2)
    tokens = _log(rng, 1, 8192)
    while tokens * top_k * n * k > 8192 * 4096 * 14336 / 2:
        tokens = (tokens + 1) // 2
    return dict(op=op, tokens=tokens, experts=experts, top_k=top_k, n=n, k=k, kind=kind, act=act, gather=rng.random() < 0.5,
                skew=rng.choice([0.0, 0.4, 1.0]))


# ------------------------------------------------------------------ what a case holds

def _counts(case):
    """Tokens of each expert, the most popular first: shares that fall as a power of the rank, at most every token."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    share = [(i + 1.0) ** -case["skew"] for i in range(e)]
    total = sum(share)
    counts = [min(t, int(t * k * s / total)) for s in share]
    left, i = t * k - sum(counts), 0
    while left:
        if counts[i % e] < t:
            counts[i % e] += 1
            left -= 1
        i += 1
    return counts


def _padding(case):
    """Whether each row of a route case is padding."""
    return [case["padded"] and t % 16 == 15 for t in range(case["tokens"])]


def work(case):
    t = case["tokens"]
    if case["op"] == "route":
        e, k = case["experts"], case["top_k"]
        live = t - sum(_padding(case))
        return {"bytes": live * e * (2 if case["logits"] == "bf16" else 4) + live * k * 16 + 4 * (e + 1),
                "flops": live * (e + 4 * k)}
    if case["op"] == "norm":
        h, rows = case["hidden"], max(1, case["top_k"]) * t
        gate = {"none": 0, "channel": 2 * h, "token": 2 * t, "full": 2 * t * h}[case["gate"]]
        return {"bytes": 2 * h * (rows + 2 * t + (t if case["pre"] else 0)) + gate
                + 4 * h * (case["post"] + case["pre"]) + (8 * rows if case["top_k"] else 0),
                "flops": h * (2 * rows + t * (3 + 4 * case["post"] + 4 * case["pre"]))}
    counts = _counts(case)
    m, n, k = sum(counts), case["n"], case["k"]
    used = sum(c > 0 for c in counts)
    x = min(m, t) if case["gather"] else m
    weights = used * n * (2 * k if case["kind"] == "bf16" else k + 4)
    return {"bytes": weights + 2 * x * k + 2 * m * (n // 2 if case["act"] else n), "flops": 2 * m * n * k}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def i32(v):
        return torch.as_tensor(v, dtype=torch.int32).to(DEV)

    st, t = dict(case=case), case["tokens"]
    if case["op"] == "route":
        e, k = case["experts"], case["top_k"]
        logits = 2.0 * normal(t, e) + normal(e)                  # some experts are liked by every token
        st.update(logits=logits.to(torch.bfloat16) if case["logits"] == "bf16" else logits,
                  bias=0.2 * normal(e) if case["bias"] else None,
                  positions=i32([-1 if p else 100 + i for i, p in enumerate(_padding(case))]) if case["padded"] else None)
        if own:
            lib, serve = _library()
            st["routing"] = serve.routing(lib, t, e, k)
        st.update(weights=torch.zeros(t, k, device=DEV), experts=i32([[0] * k] * t), places=i32([[0] * k] * t),
                  rows=i32([0] * (t * k)), offsets=i32([0] * (e + 1)))
    elif case["op"] == "experts":
        e, n, k = case["experts"], case["n"], case["k"]
        counts, ident = _counts(case), torch.randperm(e, generator=h).tolist()
        of = [0] * e
        for c, i in zip(counts, ident):
            of[i] = c
        rows = torch.cat([torch.randperm(t, generator=h)[:c].sort().values for c in of])
        m = int(rows.numel())
        w = torch.empty(e, n, k, dtype=torch.bfloat16, device=DEV)
        scales = None
        if case["kind"] == "bf16":
            w.normal_(generator=g).mul_(k ** -0.5)
        else:
            w.normal_(generator=g).mul_(60.0)                    # stored as value / scale
            w, scales = w.to(E4M3), (1 + 0.2 * normal(e, n).clamp(-2, 2)) / (60.0 * k ** 0.5)
        st.update(w=w, scales=scales, x=normal(t if case["gather"] else m, k).to(torch.bfloat16),
                  rows=rows.to(torch.int32).to(DEV) if case["gather"] else None,
                  offsets=i32([sum(of[:i]) for i in range(e + 1)]),
                  out=torch.zeros(m, n // 2 if case["act"] else n, dtype=torch.bfloat16, device=DEV))
    else:
        hid, k = case["hidden"], case["top_k"]
        shape = {"none": None, "channel": (hid,), "token": (t, 1), "full": (t, hid)}[case["gate"]]
        st.update(x=normal(t * max(1, k), hid).to(torch.bfloat16), h=3.0 * normal(t, hid), places=None, weights=None,
                  post=1 + 0.1 * normal(hid) if case["post"] else None, pre=1 + 0.1 * normal(hid) if case["pre"] else None,
                  gate=None if shape is None else torch.sigmoid(normal(*shape)).to(torch.bfloat16),
                  h_out=torch.zeros(t, hid, dtype=torch.bfloat16, device=DEV),
                  out=torch.zeros(t, hid, dtype=torch.bfloat16, device=DEV) if case["pre"] else None)
        st["h"] = st["h"].to(torch.bfloat16)
        if k:
            st.update(places=i32(torch.randperm(t * k, generator=h).view(t, k)), weights=torch.softmax(normal(t, k), -1))
    return st


# ------------------------------------------------------------------ the framework's calls

_kept = {}                    # what a program keeps for its lifetime: the library's handle, the products' workspace


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
    if c["op"] == "route":
        r = st["routing"]
        serve.route(lib, st["logits"], r, scoring=c["scoring"], bias=st["bias"], renormalise=c["renorm"], scale=1.0,
                    positions=st["positions"])
        return r.weights, r.experts, r.places, r.rows, r.offsets
    if c["op"] == "experts":
        if "ws" not in _kept:
            _kept["ws"] = serve.expert_workspace(lib)
        serve.expert_matmul(lib, st["w"], st["x"], st["offsets"], st["out"], _kept["ws"], scales=st["scales"],
                            rows=st["rows"], silu=c["act"])
        return st["out"]
    serve.block_norm(lib, st["h"], st["x"], st["h_out"], out=st["out"], places=st["places"], weights=st["weights"],
                     post=st["post"], gate=st["gate"], scale=c["scale"], pre=st["pre"], eps=1e-5)
    return (st["h_out"], st["out"]) if c["pre"] else st["h_out"]


# ------------------------------------------------------------------ the plain forms

def _plain_route(st):
    c = st["case"]
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    logits = st["logits"].float()
    if c["scoring"] == "softmax":
        score = logits
    else:
        score = 1 / (1 + torch.exp(-logits.double()))
        if c["bias"]:
            score = score + st["bias"].double()
    ids = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = logits.gather(1, ids)
    if c["scoring"] == "softmax":
        p = torch.exp(chosen - logits.amax(1, keepdim=True))
        w = p / (p if c["renorm"] else torch.exp(logits - logits.amax(1, keepdim=True))).sum(1, keepdim=True)
    else:
        w = 1 / (1 + torch.exp(-chosen))
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
    live = torch.ones(t, 1, dtype=torch.bool, device=DEV) if st["positions"] is None else st["positions"].view(t, 1) >= 0
    st["weights"].copy_(torch.where(live, w, 0.0))
    st["experts"].copy_(torch.where(live, ids, -1))
    flat = torch.where(live, ids, e).flatten()
    order = torch.sort(flat, stable=True).indices                # slots by expert, padding behind all
    at = torch.empty_like(order)
    at[order] = torch.arange(t * k, device=DEV)
    st["places"].copy_(torch.where(live, at.view(t, k), -1))
    st["offsets"].copy_((flat[:, None] < torch.arange(e + 1, device=DEV)).sum(0))
    st["rows"].copy_(torch.where(torch.arange(t * k, device=DEV) < st["offsets"][e], order // k, st["rows"]))
    return st["weights"], st["experts"], st["places"], st["rows"], st["offsets"]


def _plain_experts(st):
    c = st["case"]
    at = st["offsets"].tolist()
    x = st["x"] if st["rows"] is None else st["x"][st["rows"].long()]
    for i in range(c["experts"]):
        lo, hi = at[i], at[i + 1]
        if lo == hi:
            continue
        y = x[lo:hi].float() @ st["w"][i].float().T
        if c["kind"] == "fp8":
            y = y * st["scales"][i]
        if c["act"]:
            gate, up = y[:, :c["n"] // 2], y[:, c["n"] // 2:]
            y = gate / (1 + torch.exp(-gate)) * up
        st["out"][lo:hi] = y.to(torch.bfloat16)
    return st["out"]


def _plain_norm(st):
    c = st["case"]
    x = st["x"].float()
    y = x if st["places"] is None else (x[st["places"].long()] * st["weights"][:, :, None]).sum(1)
    if c["post"]:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5) * st["post"]
    if st["gate"] is not None:
        y = y * st["gate"].float()
    st["h_out"].copy_(st["h"].float() + c["scale"] * y)
    if not c["pre"]:
        return st["h_out"]
    h = st["h_out"].float()
    st["out"].copy_(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * st["pre"])
    return st["h_out"], st["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"route": _plain_route, "experts": _plain_experts, "norm": _plain_norm}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    f = torch.float64
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        logits = st["logits"].to(f)
        score = logits.clone() if case["scoring"] == "softmax" else torch.sigmoid(logits)
        if st["bias"] is not None:
            score += st["bias"].to(f)
        index = torch.arange(e, device=DEV)
        ids = []
        for _ in range(k):                                       # the largest, the first of equals, k times
            best = torch.where(score == score.amax(1, keepdim=True), index, e).amin(1)
            ids.append(best)
            score[torch.arange(t, device=DEV), best] = -math.inf
        ids = torch.stack(ids, 1)
        p = torch.softmax(logits, 1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
        w = p.gather(1, ids)
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        live = torch.tensor([not p for p in _padding(case)], device=DEV)
        w[~live], ids[~live] = 0, -1
        places, rows, offsets = torch.full((t, k), -1, device=DEV), st["rows"].clone(), [0]
        for i in range(e):
            slot = (ids.flatten() == i).nonzero()[:, 0]
            lo, hi = offsets[-1], offsets[-1] + int(slot.numel())
            places.view(-1)[slot] = torch.arange(lo, hi, device=DEV)
            rows[lo:hi] = (slot // k).to(torch.int32)
            offsets.append(hi)
        return w, ids.to(torch.int32), places.to(torch.int32), rows, torch.tensor(offsets, dtype=torch.int32, device=DEV)
    if case["op"] == "experts":
        out = torch.zeros(st["out"].shape, dtype=f, device=DEV)
        at = st["offsets"].tolist()
        for i in range(case["experts"]):
            rows = torch.arange(at[i], at[i + 1], device=DEV)
            if not rows.numel():
                continue
            w = st["w"][i].to(f)
            if st["scales"] is not None:
                w = w * st["scales"][i].to(f)[:, None]
            y = torch.einsum("nk,mk->mn", w, st["x"][rows if st["rows"] is None else st["rows"][rows].long()].to(f))
            if case["act"]:
                gate, up = y.chunk(2, 1)
                y = torch.nn.functional.silu(gate) * up
            out[rows] = y
        return out
    x, hid = st["x"].to(f), case["hidden"]
    y = x
    if case["top_k"]:
        y = torch.einsum("tj,tjh->th", st["weights"].to(f), x[st["places"].long()])
    if case["post"]:
        y = y / torch.sqrt((y * y).sum(1, keepdim=True) / hid + 1e-5) * st["post"].to(f)
    if st["gate"] is not None:
        y = y * st["gate"].to(f)
    h = st["h"].to(f) + case["scale"] * y
    if not case["pre"]:
        return h
    # the norm before the next block reads the residual as it is kept, in bf16
    kept = h.to(torch.bfloat16).to(f)
    return h, kept / torch.sqrt((kept * kept).sum(1, keepdim=True) / hid + 1e-5) * st["pre"].to(f)
