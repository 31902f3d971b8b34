"""The operators of a block with experts on the GPU where sizes, ranges and values go to their limits, against their 64-bit
forms (tests/expert_cases.py)."""
import pytest
import torch

import expert_cases as C
from test_experts_gpu import DEV, L, gen, route_case, run, within, ws  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ routing

@pytest.mark.parametrize("tokens", [1 << 24, (1 << 24) - 4321])
def test_routes_of_an_expert_that_nearly_every_token_takes(L, tokens):
    """The most tokens that a call may have: a CTA's share of one expert is over 100000 slots."""
    from paia_gemv import serve
    logits = torch.zeros(tokens, 2, device=DEV)
    logits[999::1000, 1] = 1.0
    r = serve.routing(L, tokens, 2, 1)
    r.rows.fill_(-9)
    serve.route(L, logits, r)
    other = logits[:, 1] > 0
    n = int((~other).sum())
    assert r.offsets.tolist() == [0, n, tokens]
    assert torch.equal(r.experts[:, 0], other.int())
    assert torch.equal(r.rows, torch.cat([(~other).nonzero()[:, 0], other.nonzero()[:, 0]]).int())
    places = torch.where(other, n + other.cumsum(0) - 1, (~other).cumsum(0) - 1)
    assert torch.equal(r.places[:, 0], places.int())
    assert bool((r.weights == 1).all())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,top_k", [(4737, 64, 8), (5003, 17, 3), (20011, 100, 6), (9000, 1024, 2)])
def test_routes_of_several_tokens_per_warp(L, scoring, tokens, experts, top_k):
    """Two launches in which a warp counts through a run of tokens, the last runs shorter, padding among them."""
    g = gen(tokens)
    logits = 2 * torch.randn(tokens, experts, generator=g, device=DEV) + 2 * torch.randn(experts, generator=g, device=DEV)
    pos = torch.arange(tokens, device=DEV, dtype=torch.int32)
    pos[5::11] = -1
    pos[600:700] = -1
    route_case(L, logits, top_k, scoring=scoring)
    route_case(L, logits.to(C.BF16), top_k, scoring=scoring, positions=pos)


def routes_far_below_zero(L, logits, bias=None):
    """Order as C.route has it; shares of the sum by logarithms (e^-l alone is infinite in 64 bits from l = -710 on)."""
    from paia_gemv import serve
    r = serve.routing(L, *logits.shape, 8)
    serve.route(L, logits, r, scoring="sigmoid", bias=bias)
    ids = C.route(logits, 8, scoring="sigmoid", bias=bias)[1]
    assert torch.equal(r.experts.cpu().long(), ids)
    chosen = logits.cpu().double().gather(1, ids)
    want = torch.softmax(torch.nn.functional.logsigmoid(chosen), 1)
    want[torch.isneginf(chosen).all(1)] = 0
    # exponentials of differences up to 200: 2^-16 of a weight (of smaller ones: nothing that fp32 holds)
    assert bool(((r.weights.cpu().double() - want).abs() <= 2.0 ** -16 * want + 1e-37).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("level", [-85.0, -95.0, -200.0, -700.0])
def test_sigmoid_weights_of_logits_far_below_zero(L, level, dtype):
    """s itself leaves fp32's range; over the sum of the chosen it is an ordinary weight."""
    g = gen(7)
    logits = (level + 3 * torch.randn(20, 64, generator=g, device=DEV)).clamp(max=-80.0).to(dtype)
    logits[11] = -float("inf")
    logits[12, 3] = 1.0
    routes_far_below_zero(L, logits)
    route_case(L, logits, 8, scoring="sigmoid", scale=3.0, renormalise=False)
    bias = torch.where(torch.arange(64, device=DEV) % 4 == 0, 2.0, 0.0)      # the chosen are not those of the largest s
    near = torch.where(torch.arange(64, device=DEV) % 4 == 0, logits.float(), torch.randn(20, 64, generator=g, device=DEV))
    routes_far_below_zero(L, near.to(dtype), bias)


# ------------------------------------------------------------------ products

@pytest.mark.parametrize("tokens", [3, 100, 200])
@pytest.mark.parametrize("xe,we,size", [(-120, 115, 64.0), (120, -147, 0.02), (-126, 120, 100.0), (126, -149, 1.0)])
def test_magnitudes_beyond_fp32_half_way(L, ws, xe, we, size, tokens):
    """Rows of x and scales of W so far apart that a sum of W's stored values, times either alone, would leave fp32's range."""
    from paia_gemv import serve
    g = gen(15)
    q = (size * torch.randn(1, 64, 128, generator=g, device=DEV)).clamp(-448, 448).to(C.E4M3)
    s = torch.full((1, 64), 2.0 ** we, device=DEV)
    x = (torch.randn(tokens, 128, generator=g, device=DEV).clamp(-3, 3).double() * 2.0 ** xe).to(C.BF16)
    out = torch.zeros(tokens, 64, dtype=C.BF16, device=DEV)
    off = C.groups([tokens], DEV)
    serve.expert_matmul(L, q, x, off, out, ws, scales=s)
    want, bound = C.matmul(q.to(C.F64) * s.to(C.F64)[:, :, None], x, off)
    if tokens > 64:
        # W meets x as bf16, and sums of x with what W stores are fp32's: where products of one sign (or those whose order is
        # the kernel's own) may add up to 2^128, which they do for x of 2^126, a sum may be infinite or NaN
        fits = x.to(C.F64).abs() @ q[0].to(C.F64).abs().T < 2.0 ** 128
        assert bool(fits.all()) == (xe < 126)
        out, want, bound = out[fits], want[fits], bound[fits]
    within(out, want, bound)


@pytest.mark.parametrize("tokens", [3, 60, 100, 200])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("gather", [False, True])
def test_every_finite_x(L, ws, kind, tokens, gather):
    """Ones on the diagonal of W: out is x to the bit, with rows of values from bf16's smallest to its largest."""
    from paia_gemv import serve
    g = gen(tokens)
    x = torch.randint(0, 0x7F80, (tokens, 512), generator=g, device=DEV)
    x = (x | torch.randint(0, 2, x.shape, generator=g, device=DEV) << 15).to(torch.int16).view(C.BF16)
    x[1, 100:] = 0
    w = torch.eye(512, device=DEV)[None].to(C.E4M3 if kind == "fp8" else C.BF16)
    s = torch.ones(1, 512, device=DEV) if kind == "fp8" else None
    rows = torch.randperm(tokens, generator=g, device=DEV).to(torch.int32) if gather else None
    out = torch.full((tokens, 512), 7.0, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, C.groups([tokens], DEV), out, ws, scales=s, rows=rows)
    assert torch.equal(out, x if rows is None else x[rows.long()])


@pytest.mark.parametrize("tokens", [3, 100, 200])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_infinities_and_nan_as_the_formula_has_them(L, ws, kind, tokens):
    """An infinity in x takes the sign of the weight that it meets; with a weight of zero, or another of the other sign, NaN."""
    from paia_gemv import serve
    g = gen(16)
    w, s, values = C.weights(1, 128, 256, kind, g, DEV)
    w[0, 5, 7] = 0
    values[0, 5, 7] = 0
    x = torch.randn(tokens, 256, generator=g, device=DEV).to(C.BF16)
    inf = float("inf")
    x[0, 7], x[1, 9], x[2, 3], x[2, 200] = inf, -inf, inf, -inf
    x[tokens - 1, 255] = float("nan") if tokens > 3 else x[tokens - 1, 255]
    out = torch.zeros(tokens, 128, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, C.groups([tokens], DEV), out, ws, scales=s)
    want = x.to(C.F64) @ values[0].T
    assert bool(torch.isinf(want[:2]).any()) and bool(torch.isnan(want[:3]).any())
    endless = torch.isinf(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[endless].to(C.F64), want[endless])
    fine = torch.isfinite(x.float()).all(1)
    _, bound = C.matmul(values, torch.where(fine[:, None], x, 0.0), C.groups([tokens], DEV))
    within(out[fine], want[fine], bound[fine])


@pytest.mark.parametrize("counts", [[5, 0, 9, 40], [100], [200, 130]], ids=str)
@pytest.mark.parametrize("n,k", [(200, 48), (200, 528), (64, 16384)])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_small_elements_whose_large_neighbours_meet_no_weight(L, ws, counts, n, k, silu, gather):
    """e4m3 rows of W that are zero wherever x is large: the sums are those of what lies 2^-30 to 2^-60 below."""
    from paia_gemv import serve
    g, m = gen(k + n), sum(counts)
    e, off = len(counts), C.groups(counts, DEV)
    w, s, values = C.weights(e, n, 2 * k, "fp8", g, DEV)
    w, values = w[:, :, k:], values[:, :, k:]
    w[:, 1::2, ::3] = 0
    values[:, 1::2, ::3] = 0
    x = torch.randn(m, 2 * k, generator=g, device=DEV)[:, :k]
    x = (x * 2.0 ** (-30 * torch.rand(m, k, generator=g, device=DEV) - 10)).to(C.BF16)
    x[:, ::3] = (2.0 ** 20 * torch.randn(x[:, ::3].shape, generator=g, device=DEV)).to(C.BF16)
    x[2] = 0
    big = torch.zeros(m, 2 * k, dtype=C.BF16, device=DEV)
    big[:, :k] = x
    rows = torch.randint(0, m, (m,), generator=g, device=DEV).to(torch.int32) if gather else None
    out = torch.full((m, n // 2 if silu else n), 7.0, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, big[:, :k], off, out, ws, scales=s, rows=rows, silu=silu)
    values = values.contiguous()
    at = off.tolist()
    for i in range(e):
        lo, hi = at[i], at[i + 1]
        xx = (x[lo:hi] if rows is None else x[rows[lo:hi].long()]).to(C.F64)
        y = xx @ values[i].T
        # C.matmul's roundings, and those of up to K products that are added one after another
        d = (xx.abs() @ values[i].abs().T) * (k / 8 + 64 + k / 2) * C.F32 + 4 * C.F32 * y.abs()
        if silu:
            (gate, up), (dg, du) = y.chunk(2, 1), d.chunk(2, 1)
            half = torch.sigmoid(gate)
            y = gate * half * up
            d = 1.1 * dg * (up.abs() + du) + (gate * half).abs() * du + y.abs() * (8 + gate.abs()) * 2 * C.F32
        within(out[lo:hi], y, d * (1 + C.HALF_BF16) + C.HALF_BF16 * y.abs() + 1e-38)
    again = torch.zeros_like(out)
    serve.expert_matmul(L, w, big[:, :k], off, again, ws, scales=s, rows=rows, silu=silu)
    assert torch.equal(out, again) and L.device_error() == 0


@pytest.mark.parametrize("silu", [False, True])
def test_captured_calls_follow_what_x_holds(L, silu):
    """e4m3, few rows: a captured call on rows of ordinary values, then of elements that only meet zeros of W beside larger ones,
    infinities among them, then ordinary ones again: to the bit as calls of their own."""
    from paia_gemv import serve
    g = gen(18)
    space = serve.expert_workspace(L)
    counts = [7, 0, 30, 1]
    w, s, values = C.weights(4, 96, 512, "fp8", g, DEV)
    w[:, 1::2, :8] = 0
    off, m = C.groups(counts, DEV), sum(counts)
    plain = torch.randn(m, 512, generator=g, device=DEV).to(C.BF16)
    wide = (plain.float() * 2.0 ** -30).to(C.BF16)
    wide[:, :8] = 3.0
    endless = wide.clone()
    endless[::3, 100] = float("inf")
    x, out = plain.clone(), torch.zeros(m, 48 if silu else 96, dtype=C.BF16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serve.expert_matmul(L, w, x, off, out, space, scales=s, silu=silu)
    for now in (plain, wide, endless, plain):
        x.copy_(now)
        graph.replay()
        alone = torch.zeros_like(out)
        serve.expert_matmul(L, w, now, off, alone, space, scales=s, silu=silu)
        assert torch.equal(out.view(torch.int16), alone.view(torch.int16))
        assert bool(torch.isfinite(out).all()) == (now is not endless)
        if now is wide:                                          # rows that are zero at the large elements
            assert bool((out[:, 1::2] != 0).any()) and out[:, 1::2].abs().max() < 2.0 ** -20


# More than two rounds of tiles: runs of K that end inside tiles, then whole tiles, three parts and more for every CTA (pair).
# Units of K: one, three with the last one short, seven.
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("kind,k", [("bf16", 64), ("bf16", 168), ("bf16", 448), ("fp8", 128), ("fp8", 368), ("fp8", 896)])
@pytest.mark.parametrize("counts,n", [([300, 0, 257, 130], 10496), ([150, 513, 0, 1, 290, 190], 8192), ([256, 256], 19200)],
                         ids=str)
def test_many_tiles_of_large_blocks(L, ws, counts, n, kind, k, gather, silu):
    """Pairs of CTAs, tile after tile."""
    a = run(L, ws, counts, n, k, kind, silu, gather, tokens=700 if gather else None, seed=k)
    assert torch.equal(a, run(L, ws, counts, n, k, kind, silu, gather, tokens=700 if gather else None, seed=k))
    assert not ws.buffer[:1280].any()


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("kind,k", [("bf16", 168), ("bf16", 448), ("fp8", 368), ("fp8", 896)])
@pytest.mark.parametrize("counts,n", [([1] * 40, 1536), ([9, 0, 17, 1, 30, 2] * 6, 1664), ([60, 64, 3, 50] * 2, 7296)], ids=str)
def test_many_tiles_of_small_blocks(L, ws, counts, n, kind, k, gather, silu):
    """Single CTAs, tile after tile (e4m3: as split terms)."""
    a = run(L, ws, counts, n, k, kind, silu, gather, tokens=100 if gather else None, seed=k)
    assert torch.equal(a, run(L, ws, counts, n, k, kind, silu, gather, tokens=100 if gather else None, seed=k))
    assert not ws.buffer[:1280].any()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("k", [1040, 4096])
def test_one_round_of_whole_tiles(L, ws, kind, k):
    """Tiles that nearly fill a round are taken whole, each from another place of K on."""
    run(L, ws, [1] * 8, 2048, k, kind, silu=True, gather=True, tokens=1)
    run(L, ws, [3, 1, 0, 2, 2, 1, 1, 1, 5], 2048, k, kind)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("experts,rows", [(256, 8), (96, 21), (64, 40)])
def test_small_blocks_of_converted_weights(L, ws, experts, rows, gather, silu):
    """e4m3 rows whose terms would not fit the workspace: blocks of 16 to 128 tokens meet converted weights, an odd number of
    units of K two by two."""
    counts = [rows + (i % 5) - 2 for i in range(experts)]
    counts[3], counts[4] = 0, counts[3] + counts[4]
    k = 7024                                                     # 55 units
    assert sum(counts) * (4 * k + 4) > 48 << 20
    a = run(L, ws, counts, 144, k, "fp8", silu, gather, tokens=300 if gather else None)
    assert torch.equal(a, run(L, ws, counts, 144, k, "fp8", silu, gather, tokens=300 if gather else None))


# ------------------------------------------------------------------ norms

def test_block_of_no_places_is_refused(L):
    """Places without a column are no call without places, which adds x's own rows."""
    from paia_gemv import serve
    h, x = torch.zeros(4, 64, dtype=C.BF16, device=DEV), torch.ones(4, 64, dtype=C.BF16, device=DEV)
    places, weights = torch.zeros(4, 0, dtype=torch.int32, device=DEV), torch.zeros(4, 0, device=DEV)
    with pytest.raises(ValueError, match="places"):
        serve.block_norm(L, h, x, h, places=places, weights=weights)
    assert not h.any()


def test_norms_of_nearly_2_31_rows(L):
    """The most rows that an int counts (one row of h for all of them): the last are reached, and nothing behind."""
    from paia_gemv import serve
    tokens = 2 ** 31 - 1
    g = gen(17)
    h = torch.randn(1, 8, generator=g, device=DEV).to(C.BF16)
    pre = 1 + 0.1 * torch.randn(8, generator=g, device=DEV)
    small = torch.zeros(1, 8, dtype=C.BF16, device=DEV)
    serve.block_norm(L, h, out=small, pre=pre)
    within(small, *C.norm(h, pre))
    out = torch.full((tokens + 1, 8), 7.0, dtype=C.BF16, device=DEV)
    serve.block_norm(L, h.expand(tokens, 8), out=out[:tokens], pre=pre)
    assert bool((out[tokens] == 7.0).all())
    for piece in out[:tokens].split(1 << 28):
        assert bool((piece == small).all())
