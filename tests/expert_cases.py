"""Plain 64-bit forms of the operators of a block with experts (include/paia_gemv.h) with bounds for what the kernels may be
off, and builders of their inputs. Shared by the GPU tests; runs on any device."""
import torch

BF16, E4M3, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float64
HALF_BF16 = 2.0 ** -8                              # half a step, relative to the value
F32 = 2.0 ** -23                                   # one fp32 step: an MMA may cut off where it adds


def groups(counts, device):
    """offsets of groups of these sizes, one behind the other."""
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device=device)


def weights(e, n, k, kind, g, device):
    """(stored weights, scales or None, the values they stand for in 64 bits)"""
    if kind == "bf16":
        w = torch.randn(e, n, k, generator=g, device=device).mul_(k ** -0.5).to(BF16)
        return w, None, w.to(F64)
    q = torch.randn(e, n, k, generator=g, device=device).mul_(60.0).clamp(-448, 448).to(E4M3)
    s = (1 + 0.2 * torch.randn(e, n, generator=g, device=device)).abs() / (60 * k ** 0.5)
    return q, s, q.to(F64) * s.to(F64)[:, :, None]


def matmul(values, x, offsets, rows=None, silu=False, split=False):
    """(out, bound) for rows 0 .. offsets[-1] - 1: fp32 sums of K exact products (one step for every 8 of them and 64 for the
    joins), with split terms 2^-34 of a row's largest in each x, a scale's and a product's rounding, silu's quotient and
    exponential, and the output's rounding."""
    at = offsets.tolist()
    n, k = values.shape[1:]
    y = torch.zeros(at[-1], n, dtype=F64, device=x.device)
    d = torch.zeros_like(y)
    for e in range(values.shape[0]):
        lo, hi = at[e], at[e + 1]
        if lo == hi:
            continue
        xx = (x[lo:hi] if rows is None else x[rows[lo:hi].long()]).to(F64)
        y[lo:hi] = xx @ values[e].T
        d[lo:hi] = (xx.abs() @ values[e].abs().T) * (k / 8 + 64) * F32 + 4 * F32 * y[lo:hi].abs()
        if split:
            d[lo:hi] += 2.0 ** -34 * xx.abs().amax(1, keepdim=True) * values[e].abs().sum(1)
    if silu:
        g, u = y.chunk(2, 1)
        dg, du = d.chunk(2, 1)
        s = torch.sigmoid(g)
        y = g * s * u
        # the quotient's two roundings, e^-g to 2 steps and |g| 2^-23 of it
        d = 1.1 * dg * (u.abs() + du) + (g * s).abs() * du + y.abs() * (8 + g.abs()) * 2 * F32
    return y, d * (1 + HALF_BF16) + HALF_BF16 * y.abs() + 1e-38


def block(h, x, places=None, weights=None, post=None, gate=None, scale=1.0, eps=1e-5):
    """(h_out, bound): sums over top_k in fp32, a sum of squares of up to 32768 elements (each thread's 64, then a tree: 2^-17
    of the root covers it), three products, the output's rounding."""
    xx = x.to(F64)
    if places is None:
        y, mag = xx[:h.shape[0]], xx[:h.shape[0]].abs()
        k = 0
    else:
        w = torch.where(places >= 0, weights.to(F64), 0.0)[:, :, None]
        rows = xx[places.clamp(min=0).long()]
        y, mag, k = (rows * w).sum(1), (rows * w).abs().sum(1), places.shape[1]
    d = mag * (k + 2) * F32
    if post is not None:
        r = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        # what a row's sums are off moves its root too: by at most the relative error of its largest elements' sum
        rel = (d.square().sum(-1, keepdim=True).sqrt() / y.norm(dim=-1, keepdim=True).clamp(min=1e-30)).clamp(max=1.0)
        y = y * r * post.to(F64)
        d = (d * r * post.to(F64).abs()) + y.abs() * (2.0 ** -17 + rel)
    if gate is not None:
        y, d = y * gate.to(F64), d * gate.to(F64).abs()
    out = h.to(F64) + scale * y
    d = abs(scale) * (d + 4 * F32 * y.abs()) + F32 * out.abs()
    return out, d * (1 + HALF_BF16) + HALF_BF16 * out.abs() + 1e-38


def norm(h, pre, eps=1e-5):
    y = h.to(F64)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * pre.to(F64)
    return y, y.abs() * (2.0 ** -17 + HALF_BF16) + 1e-38


def route(logits, top_k, scoring="softmax", bias=None, renormalise=True, scale=1.0, positions=None):
    """(weights in 64 bits, ids, places, rows, offsets) of all tokens: by falling score, the first of equals, NaN last."""
    t, e = logits.shape
    l = logits.to(F64)
    score = l.clone() if scoring == "softmax" else 1 / (1 + torch.exp(-l))
    if bias is not None:
        score = score + bias.to(F64)
    nan = torch.isnan(score).cpu()
    order = torch.sort(torch.where(nan, -torch.inf, score.cpu()), dim=1, descending=True, stable=True).indices
    last = torch.sort(nan.gather(1, order).int(), dim=1, stable=True).indices
    ids = order.gather(1, last)[:, :top_k].clone()
    chosen = l.cpu().gather(1, ids)
    if scoring == "softmax":
        top = chosen[:, :1]
        p = torch.exp(chosen - top)
        w = p / (p if renormalise else torch.exp(l.cpu() - top)).sum(1, keepdim=True)
        w = torch.where(torch.isneginf(top), 0.0, w)
    else:
        w = 1 / (1 + torch.exp(-chosen))
        if renormalise:
            total = w.sum(1, keepdim=True)
            w = torch.where(total == 0, 0.0, w / total)
    w = w * scale
    if positions is not None:
        dead = positions.cpu() < 0
        w[dead], ids[dead] = 0, -1
    flat = ids.flatten()
    slots = torch.sort(torch.where(flat < 0, e, flat), dim=0, stable=True).indices[:int((flat >= 0).sum())]
    places = torch.full((t * top_k,), -1)
    places[slots] = torch.arange(len(slots))
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(flat[flat >= 0], minlength=e).cumsum(0)])
    return w, ids, places.view(t, top_k), slots // top_k, offsets
