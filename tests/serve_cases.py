"""Plain 64-bit forms of the serving operators (include/paia_gemv.h) with bounds for what the kernels may be off, and
builders of their inputs. Shared by the GPU tests; runs on any device."""
import math

import torch

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, E4M3: 2.0 ** -4}          # half a step, relative to the value
F32 = 2.0 ** -23                                   # one fp32 step: an MMA may cut off where it adds


def paged(lens, kv, hd, page, dtype, device, g, hnd=False, extra=3, filler=float("nan")):
    """(k, v pools [pages, page, kv, hd], table): every valid row is N(0, 1), every other row of the pools `filler`;
    table entries behind a sequence's end are absurd."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(7)).tolist()
    table = torch.full((len(lens), max(1, max(need)) + 1), 0x7FFFFFFF, dtype=torch.int32)
    shape = (pages, kv, page, hd) if hnd else (pages, page, kv, hd)
    pools = []
    for _ in range(2):
        x = torch.full(shape, filler, device=device)
        pools.append(x.transpose(1, 2) if hnd else x)
    at = 0
    for b, n in enumerate(lens):
        for c in range(need[b]):
            pg = order[at]
            at += 1
            table[b, c] = pg
            m = min(page, n - c * page)
            for x in pools:
                x[pg, :m] = torch.randn(m, kv, hd, generator=g, device=device) * (30.0 if dtype is E4M3 else 1.0)
    return pools[0].to(dtype), pools[1].to(dtype), table.to(device)


def attention(q, k, v, table, lens, scale, window=0, ks=None, vs=None):
    """(out, lse, bound of out, bound of lse) in 64 bits. The bounds add up: a score's fp32 sum of head_dim products and
    its scaling (and q in f16 next to an e4m3 cache: 2^-24 of its largest element), ex2's 2^-22, P as two bf16 (2^-16) or
    one f16 (2^-11, not below 2^-24), one fp32 step per 16 positions summed and 64 for merges, and the output's rounding."""
    f = torch.float64
    b, h, hd = q.shape
    kv, page = k.shape[2], k.shape[1]
    out = torch.zeros(b, h, hd, dtype=f, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((b, h), -math.inf, dtype=f, device=q.device)
    tol_lse = torch.zeros_like(lse)
    eight = k.dtype is E4M3
    for i, n in enumerate(lens):
        if n <= 0:
            continue
        first = max(0, n - window) if window else 0
        pos = torch.arange(first, n, device=q.device)
        rows = table[i].long()[pos // page]
        kk, vv = k[rows, pos % page].to(f), v[rows, pos % page].to(f)
        for j in range(kv):
            hs = slice(j * (h // kv), (j + 1) * (h // kv))
            c = scale * (1.0 if ks is None else float(ks[j]))
            qq = q[i, hs].to(f)
            s = c * (qq @ kk[:, j].T)
            ds = c * (hd + 16) * F32 * (qq.abs() @ kk[:, j].abs().T)
            if eight:
                ds = ds + c * 2.0 ** -24 * qq.abs().amax(-1, keepdim=True) * kk[:, j].abs().sum(-1)
            ds = ds + 4 * F32 * s.abs()
            p = torch.softmax(s, -1)
            lse[i, hs] = torch.logsumexp(s, -1)
            # one exponent's error moves its own term and the sum it is divided by
            e = ds.amax(-1, keepdim=True) * 2 + 2.0 ** -20 + (len(pos) / 16 + 64) * 2 * F32
            pe = p * (2.0 ** -11 if eight else 2.0 ** -16)
            if eight:
                pe = pe + 2.0 ** -24 * torch.exp(s.amax(-1, keepdim=True) - lse[i, hs][:, None])
            w = 1.0 if vs is None else float(vs[j])
            out[i, hs] = w * (p @ vv[:, j])
            big = p @ vv[:, j].abs()
            tol[i, hs] = w * (big * e + pe @ vv[:, j].abs()) * (1 + 2.0 ** -8) + HALF[BF16] * out[i, hs].abs() + 1e-38
            tol_lse[i, hs] = (ds.amax(-1) + 2.0 ** -20 + (len(pos) / 16 + 64) * F32
                              + 4 * F32 * (lse[i, hs].abs() + s.abs().amax(-1)))
    return out, lse, tol, tol_lse


def rope(qkv, pos, freq, heads, kv, hd, qn=None, kn=None, eps=1e-6, interleaved=False):
    """(q, k, v [tokens, ..., hd], magnitude of each element's pair) in 64 bits, every row."""
    f = torch.float64
    x = qkv.to(f).view(qkv.shape[0], heads + 2 * kv, hd).clone()
    for part, w in ((slice(0, heads), qn), (slice(heads, heads + kv), kn)):
        if w is not None:
            y = x[:, part]
            x[:, part] = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.to(f)
    half = freq.numel()
    i = torch.arange(half, device=qkv.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    ang = pos.to(f)[:, None, None] * freq
    y, mag = x.clone(), x.abs().clone()
    turn = slice(0, heads + kv)
    xa, xb = x[:, turn, a], x[:, turn, b]
    y[:, turn, a], y[:, turn, b] = xa * ang.cos() - xb * ang.sin(), xb * ang.cos() + xa * ang.sin()
    m = xa.abs() + xb.abs()
    mag[:, turn, a], mag[:, turn, b] = m, m
    return (y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]), \
        (mag[:, :heads], mag[:, heads:heads + kv], mag[:, heads + kv:])


def lora(x, a, b, adapter, base, scaling=None, ranks=None):
    """(out, bound of out) in 64 bits: fp32 sums of K and of rank products (one step each term), t kept to 2^-16, the
    output's rounding."""
    f = torch.float64
    n = b.shape[1]
    out = torch.zeros(x.shape[0], n, dtype=f, device=x.device) if base is None else base.to(f).clone()
    err = torch.zeros_like(out)
    for i in sorted(set(adapter.tolist())):
        if not 0 <= i < a.shape[0]:
            continue
        rows = (adapter == i).nonzero()[:, 0]
        r = a.shape[1] if ranks is None else min(max(int(ranks[i]), 0), a.shape[1])
        s = 1.0 if scaling is None else float(scaling[i])
        A, B, X = a[i, :r].to(f), b[i, :, :r].to(f), x[rows].to(f)
        t = X @ A.T
        dt = (X.abs() @ A.abs().T) * (x.shape[1] / 8 + 64) * F32 + t.abs() * (2.0 ** -16 + 2 * F32)
        out[rows] += s * (t @ B.T)
        err[rows] += abs(s) * (dt @ B.abs().T + (r + 8) * F32 * (t.abs() @ B.abs().T))
    return out, err * (1 + 2.0 ** -8) + F32 * out.abs() + HALF[BF16] * out.abs() + 1e-38
