"""The operators of a block with experts on the GPU against their 64-bit forms (tests/expert_cases.py), element by element:
types, group sizes from none to thousands, odd sizes, strides, NaN and infinities, bad indices, streams and graphs."""
import pytest
import torch

import expert_cases as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paia_gemv import load_lib
    lib = load_lib()
    while lib.device_error():
        pass
    return lib


@pytest.fixture(scope="module")
def ws(L):
    from paia_gemv import serve
    return serve.expert_workspace(L)


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def within(got, want, bound, what=""):
    bad = ~((got.to(C.F64) - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3].tolist(), want[bad][:3].tolist())


def run(L, ws, counts, n, k, kind, silu=False, gather=False, tokens=None, seed=0, **kw):
    from paia_gemv import serve
    g = gen(seed)
    off = C.groups(counts, DEV)
    m = sum(counts)
    w, s, values = C.weights(len(counts), n, k, kind, g, DEV)
    tokens = tokens or max(1, m)
    x = torch.randn(tokens if gather else m, k, generator=g, device=DEV).to(C.BF16)
    rows = torch.randint(0, tokens, (m,), generator=g, device=DEV).to(torch.int32) if gather else None
    out = torch.full((m, n // 2 if silu else n), 7.0, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, off, out, ws, scales=s, rows=rows, silu=silu, **kw)
    want, bound = C.matmul(values, x, off, rows, silu, split=kind == "fp8")
    within(out, want, bound, (counts, n, k, kind, silu, gather))
    assert L.device_error() == 0
    return out


# group sizes: one row; a row each; none in some; around the tiles' 16, 32, 64, 128 and 256 columns; one group only
GROUPS = [[1], [1, 0, 1, 1], [0, 5, 0, 0, 16, 17], [15, 33, 1], [64, 65, 0, 2], [128, 3, 129], [300, 7], [0, 0, 513, 40]]


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts", GROUPS, ids=str)
def test_groups(L, ws, kind, silu, gather, counts):
    run(L, ws, counts, 272, 336, kind, silu, gather, tokens=50 if gather else None)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("n,k", [(1, 16), (2, 32), (16, 64), (100, 48), (128, 128), (130, 4096), (257, 80), (384, 1040), (640, 2000)])
@pytest.mark.parametrize("tokens", [3, 200])
def test_sizes(L, ws, kind, n, k, tokens):
    run(L, ws, [tokens, 0, tokens // 2], n, k, kind)
    if n % 2 == 0:
        run(L, ws, [tokens, 0, tokens // 2], n, k, kind, silu=True, gather=True)


@pytest.mark.parametrize("k", [8, 24, 72, 136])
def test_bf16_rows_of_any_multiple_of_8(L, ws, k):
    run(L, ws, [2, 9], 64, k, "bf16")
    run(L, ws, [2, 290], 64, k, "bf16", gather=True)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_many_experts(L, ws, kind):
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 4, (1024,), generator=g).tolist()
    run(L, ws, counts, 48, 64, kind, gather=True)
    run(L, ws, [0] * 1023 + [1], 48, 64, kind)
    run(L, ws, [0] * 8, 48, 64, kind)                            # nobody has a row


@pytest.mark.parametrize("kind,counts", [("bf16", [2] * 10), ("fp8", [2] * 10), ("bf16", [260, 300]), ("fp8", [260, 300])])
def test_tiles_cut_over_many_ctas(L, ws, kind, counts):
    """Few tiles of a long K: every one is summed by many CTAs, twice the same bits, and the workspace is left as it was."""
    a = run(L, ws, counts, 128, 16384, kind, seed=1)
    b = run(L, ws, counts, 128, 16384, kind, seed=1)
    assert torch.equal(a, b)
    assert not ws.buffer[:1280].any()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("tokens", [4, 300])
def test_strides(L, ws, kind, tokens):
    """Weights, scales, x and out as parts of larger tensors; what lies around out stays."""
    from paia_gemv import serve
    g, n, k = gen(5), 96, 160
    off = C.groups([tokens, 0, tokens], DEV)
    w, s, values = C.weights(6, 2 * n, 2 * k, kind, g, DEV)
    w, values = w[::2, n:, k:], values[::2, n:, k:]
    s = None if s is None else s[::2, n:]
    x = torch.randn(2 * tokens, 2 * k, generator=g, device=DEV).to(C.BF16)[:, k:]
    big = torch.full((2 * tokens + 2, 3 * n), 7.0, dtype=C.BF16, device=DEV)
    out = big[1:-1, n + 3:2 * n + 3]
    serve.expert_matmul(L, w, x, off, out, ws, scales=s)
    want, bound = C.matmul(values, x, off, split=kind == "fp8")
    within(out, want, bound)
    big[1:-1, n + 3:2 * n + 3] = 7.0
    assert bool((big == 7.0).all())


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("tokens", [3, 200])
def test_rows_of_no_expert_stay(L, ws, kind, tokens):
    from paia_gemv import serve
    g = gen(6)
    off = C.groups([tokens, 1], DEV)
    w, s, values = C.weights(2, 64, 128, kind, g, DEV)
    x = torch.randn(tokens + 9, 128, generator=g, device=DEV).to(C.BF16)
    out = torch.full((tokens + 9, 64), 7.0, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, off, out, ws, scales=s)
    want, bound = C.matmul(values, x, off, split=kind == "fp8")
    within(out[:tokens + 1], want, bound)
    assert bool((out[tokens + 1:] == 7.0).all())


def test_small_terms_beside_a_large_one(L, ws):
    """fp32 sums: 4095 products of 2^-15 of the largest one add up to an eighth of it, in every path."""
    from paia_gemv import serve
    k = 4096
    for kind, counts in (("bf16", [3]), ("fp8", [3]), ("bf16", [200]), ("fp8", [100]), ("fp8", [200])):
        w = torch.full((1, 128, k), 2.0 ** -7, device=DEV)
        w[:, :, 0] = 256.0
        s = torch.ones(1, 128, device=DEV) if kind == "fp8" else None
        x = torch.ones(sum(counts), k, dtype=C.BF16, device=DEV)
        out = torch.zeros(sum(counts), 128, dtype=C.BF16, device=DEV)
        serve.expert_matmul(L, w.to(C.E4M3 if kind == "fp8" else C.BF16), x, C.groups(counts, DEV), out, ws, scales=s)
        want = 256 + (k - 1) * 2.0 ** -7
        assert bool(((out.double() - want).abs() <= want * C.HALF_BF16).all()), (kind, counts, out[0, 0].item())


@pytest.mark.parametrize("tokens", [2, 100, 200])
def test_every_e4m3_code(L, ws, tokens):
    """Each of the 256 codes as a weight, alone in its row: exact, NaN where it is NaN."""
    from paia_gemv import serve
    w = torch.zeros(1, 256, 256, dtype=torch.uint8, device=DEV)
    i = torch.arange(256, device=DEV)
    w[0, i, i] = i.to(torch.uint8)
    x = torch.full((tokens, 256), 0.5, dtype=C.BF16, device=DEV)
    out = torch.zeros(tokens, 256, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, C.groups([tokens], DEV), out, ws, scales=torch.ones(1, 256, device=DEV))
    want = w[0, i, i].view(C.E4M3).float() * 0.5
    assert bool(((out.float() == want) | (torch.isnan(out.float()) & torch.isnan(want))).all())
    assert torch.isnan(out.float()).sum().item() == 2 * tokens


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("tokens", [5, 100, 300])
@pytest.mark.parametrize("gather", [False, True])
def test_nan_and_infinity_reach_their_rows_alone(L, ws, kind, tokens, gather):
    from paia_gemv import serve
    g = gen(8)
    off = C.groups([tokens, tokens], DEV)
    w, s, values = C.weights(2, 128, 256, kind, g, DEV)
    x = torch.randn(2 * tokens, 256, generator=g, device=DEV).to(C.BF16)
    x[1, 7], x[tokens + 2, 255], x[3, 0] = float("nan"), float("inf"), -float("inf")
    rows = torch.arange(2 * tokens, device=DEV, dtype=torch.int32) if gather else None
    out = torch.zeros(2 * tokens, 128, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, off, out, ws, scales=s, rows=rows)
    odd = torch.zeros(2 * tokens, dtype=torch.bool, device=DEV)
    odd[[1, 3, tokens + 2]] = True
    assert not torch.isfinite(out[odd].float()).any()
    x[odd] = 0
    want, bound = C.matmul(values, x, off, split=kind == "fp8")
    within(out[~odd], want[~odd], bound[~odd])


@pytest.mark.parametrize("exponent", [-130, -60, 0, 100])
def test_rows_of_any_magnitude(L, ws, exponent):
    """x of one row over 2^20 beside rows of other magnitudes, e4m3 weights: each row as exact as its own largest allows."""
    from paia_gemv import serve
    g = gen(9)
    off = C.groups([6], DEV)
    w, s, values = C.weights(1, 64, 128, "fp8", g, DEV)
    x = torch.randn(6, 128, generator=g, device=DEV) * 2.0 ** (-20 * torch.rand(6, 128, generator=g, device=DEV))
    x = (x.double() * 2.0 ** exponent).to(C.BF16)
    x[4] = 0
    out = torch.ones(6, 64, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, off, out, ws, scales=s)
    want, bound = C.matmul(values, x, off, split=True)
    within(out, want, bound + 2.0 ** -133)                       # bf16's smallest step
    assert not out[4].any()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("tokens", [4, 100, 300])
def test_rows_behind_the_groups_say_anything(L, ws, kind, tokens):
    """What rows holds for places of no expert is not looked at."""
    from paia_gemv import serve
    g = gen(13)
    off = C.groups([tokens, tokens], DEV) + 2
    w, s, values = C.weights(2, 64, 128, kind, g, DEV)
    x = torch.randn(tokens, 128, generator=g, device=DEV).to(C.BF16)
    rows = torch.full((2 * tokens + 5,), 0x7FFFFFFF, dtype=torch.int32, device=DEV)
    rows[2:2 * tokens + 2] = torch.arange(2 * tokens, device=DEV, dtype=torch.int32) % tokens
    out = torch.full((2 * tokens + 5, 64), 7.0, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, off, out, ws, scales=s, rows=rows)
    live = slice(2, 2 * tokens + 2)
    want, bound = C.matmul(values, x, off - 2, rows[live], split=kind == "fp8")
    within(out[live], want, bound)
    assert bool((out[:2] == 7.0).all()) and bool((out[2 * tokens + 2:] == 7.0).all())
    assert L.device_error() == 0


@pytest.mark.parametrize("xe,we", [(120, -120), (-120, 100), (60, 60)])
def test_magnitudes_that_cancel(L, ws, xe, we):
    """Rows of x and scales of W near both ends of fp32's range whose products lie well inside it."""
    from paia_gemv import serve
    g = gen(14)
    for tokens in (3, 100, 200):
        q = torch.randn(1, 64, 128, generator=g, device=DEV).to(C.E4M3)
        s = torch.full((1, 64), 2.0 ** we, device=DEV)
        x = (torch.randn(tokens, 128, generator=g, device=DEV).double() * 2.0 ** xe).to(C.BF16)
        out = torch.zeros(tokens, 64, dtype=C.BF16, device=DEV)
        off = C.groups([tokens], DEV)
        serve.expert_matmul(L, q, x, off, out, ws, scales=s)
        values = q.to(C.F64) * s.to(C.F64)[:, :, None]
        within(out, *C.matmul(values, x, off, split=True))


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("tokens", [4, 100, 300])
def test_bad_rows_and_offsets(L, ws, kind, tokens):
    """A row of x that is nowhere reads as zeros; with offsets out of order or range nothing is computed. Code 14 either way."""
    from paia_gemv import serve
    g = gen(10)
    w, s, values = C.weights(2, 64, 128, kind, g, DEV)
    x = torch.randn(tokens, 128, generator=g, device=DEV).to(C.BF16)
    rows = torch.arange(tokens, device=DEV, dtype=torch.int32)
    rows[1], rows[2] = -5, tokens
    off = C.groups([tokens, 0], DEV)
    out = torch.ones(tokens, 64, dtype=C.BF16, device=DEV)
    serve.expert_matmul(L, w, x, off, out, ws, scales=s, rows=rows)
    want, bound = C.matmul(values, x, off, split=kind == "fp8")
    keep = torch.ones(tokens, dtype=torch.bool, device=DEV)
    keep[1:3] = False
    within(out[keep], want[keep], bound[keep])
    assert not out[1:3].any()
    torch.cuda.synchronize()
    assert L.device_error() == 14 and L.device_error() == 0
    for bad in ([0, tokens + 50, tokens], [-3, 2, tokens], [tokens, 0, 2], [0, 1, tokens + 1], [-2 ** 31, 2 ** 31 - 1, 0]):
        out.fill_(7.0)
        serve.expert_matmul(L, w, x, torch.tensor(bad, dtype=torch.int32, device=DEV), out, ws, scales=s)
        torch.cuda.synchronize()
        assert L.device_error() == 14 and L.device_error() == 0, bad
        assert bool((out == 7.0).all())


def test_offsets_past_32_bits(L, ws):
    """Weights of more than 2^32 bytes, and rows of x behind 2^31 elements."""
    from paia_gemv import serve
    g = gen(11)
    w = torch.zeros(3, 32768, 32768, dtype=C.BF16, device=DEV)
    w[2, -256:] = torch.randn(256, 32768, generator=g, device=DEV).mul_(2.0 ** -7).to(C.BF16)
    x = torch.randn(70000, 32768, device=DEV, generator=g, dtype=C.BF16)
    rows = torch.tensor([69999, 0, 65536], dtype=torch.int32, device=DEV)
    out = torch.zeros(3, 32768, dtype=C.BF16, device=DEV)
    off = C.groups([0, 0, 3], DEV)
    serve.expert_matmul(L, w, x, off, out, ws, rows=rows)
    want, bound = C.matmul(w[2:, -256:].to(C.F64), x, C.groups([3], DEV), rows)
    within(out[:, -256:], want, bound)
    assert not out[:, :-256].any()


def test_streams_graphs_and_two_workspaces(L):
    """Captured calls follow the offsets of each replay; calls on two streams at once have a workspace each."""
    from paia_gemv import serve
    g = gen(12)
    spaces = [serve.expert_workspace(L) for _ in range(2)]
    off = [C.groups([5, 60, 0], DEV), C.groups([40, 1, 24], DEV)]
    w, s, values = C.weights(3, 256, 4096, "fp8", g, DEV)
    x = torch.randn(65, 4096, generator=g, device=DEV).to(C.BF16)
    outs = [torch.zeros(65, 256, dtype=C.BF16, device=DEV) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                serve.expert_matmul(L, w, x, off[i], outs[i], spaces[i], scales=s)
    torch.cuda.synchronize()
    for i in range(2):
        within(outs[i], *C.matmul(values, x, off[i], split=True))
    now = off[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serve.expert_matmul(L, w, x, now, outs[0], spaces[0], scales=s)
    for i in (1, 0, 1):
        now.copy_(off[i])
        outs[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) if i else True
        within(outs[0], *C.matmul(values, x, off[i], split=True))


# ------------------------------------------------------------------ routing

def route_case(L, logits, top_k, positions=None, **kw):
    from paia_gemv import serve
    t, e = logits.shape
    r = serve.routing(L, t, e, top_k)
    r.rows.fill_(-9)
    serve.route(L, logits, r, positions=positions, **kw)
    w, ids, places, rows, offsets = C.route(logits, top_k, positions=positions, **kw)
    assert torch.equal(r.experts.cpu().long(), ids)
    assert torch.equal(r.offsets.cpu().long(), offsets)
    assert torch.equal(r.places.cpu().long(), places)
    n = len(rows)
    assert torch.equal(r.rows[:n].cpu().long(), rows) and bool((r.rows[n:] == -9).all())
    # exponentials of differences up to 200: 2^-16 of a weight
    d = (r.weights.cpu().double() - w).abs()
    assert bool(((d <= 2.0 ** -16 * w.abs() + 1e-37) | (torch.isnan(w) & torch.isnan(r.weights.cpu()))).all())
    return r


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 64, 8), (2, 3, 3), (17, 60, 4), (33, 256, 8), (130, 129, 1),
                                                  (256, 512, 32), (257, 16, 2), (300, 1024, 10), (600, 100, 6)])
def test_routes(L, scoring, dtype, tokens, experts, top_k):
    g = gen(tokens)
    logits = (2 * torch.randn(tokens, experts, generator=g, device=DEV)).to(dtype)
    bias = 0.3 * torch.randn(experts, generator=g, device=DEV) if scoring == "sigmoid" else None
    pos = torch.arange(tokens, device=DEV, dtype=torch.int32)
    pos[3::7] = -1
    route_case(L, logits, top_k, scoring=scoring, bias=bias, scale=2.5)
    route_case(L, logits, top_k, scoring=scoring, renormalise=False, positions=pos)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routes_ties_and_far_values(L, scoring):
    """Equal logits go by index; scores that fp32 cannot tell apart go by fp64; NaN comes last, -inf has no weight."""
    g = gen(2)
    logits = torch.randint(-2, 3, (40, 96), generator=g, device=DEV).float()
    logits[5] = 0.0
    logits[6] = -float("inf")
    logits[7, ::2] = -float("inf")
    logits[8] = 30 + torch.arange(96, device=DEV) * 1e-4         # sigmoid: 1 - e^-30, apart by 1e-17
    logits[9] = 10 + torch.arange(96, device=DEV) * 1e-5         # apart by 5e-10
    logits[10] = -torch.arange(96, device=DEV) * 1.5
    logits[11] = torch.tensor([0.0, -0.0] * 48, device=DEV)
    route_case(L, logits, 8, scoring=scoring)
    route_case(L, logits, 8, scoring=scoring, renormalise=False)
    if scoring == "sigmoid":
        route_case(L, logits, 8, scoring=scoring, bias=0.25 * torch.randint(-2, 3, (96,), generator=g, device=DEV).float())
    bad = logits.clone()
    bad[2, 5:90] = float("nan")
    bad[3] = float("nan")
    from paia_gemv import serve
    r = serve.routing(L, 40, 96, 12)
    serve.route(L, bad, r, scoring=scoring)
    want = C.route(bad[2:4], 12, scoring=scoring)[1]
    assert torch.equal(r.experts[2:4].cpu().long(), want)


def test_routes_of_no_token_and_of_padding_alone(L):
    from paia_gemv import serve
    r = serve.routing(L, 0, 8, 2)
    r.offsets.fill_(5)
    serve.route(L, torch.zeros(0, 8, device=DEV), r)
    assert not r.offsets.any()
    route_case(L, torch.zeros(5, 8, device=DEV), 2, positions=torch.full((5,), -1, dtype=torch.int32, device=DEV))


def test_routes_strided_logits_and_fewer_tokens(L):
    from paia_gemv import serve
    g = gen(4)
    big = torch.randn(20, 100, generator=g, device=DEV)
    r = serve.routing(L, 50, 32, 4)
    serve.route(L, big[:, 7:39], r.first(20))
    w, ids, places, rows, offsets = C.route(big[:, 7:39], 4)
    assert torch.equal(r.experts[:20].cpu().long(), ids) and torch.equal(r.rows[:80].cpu().long(), rows)


# ------------------------------------------------------------------ norms

GATES = ["none", "channel", "token", "full"]


@pytest.mark.parametrize("hidden", [8, 264, 4096, 4104, 10000, 32768])
@pytest.mark.parametrize("tokens,top_k", [(1, 0), (1, 8), (5, 1), (37, 9), (700, 2), (700, 0)])
@pytest.mark.parametrize("variant", [0, 1, 2, 3])
def test_blocks(L, hidden, tokens, top_k, variant):
    from paia_gemv import serve
    g = gen(hidden + tokens)
    if hidden * tokens > 4096 * 700:
        tokens = 300
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)   # noqa: E731
    h, x = (3 * randn(tokens, hidden)).to(C.BF16), randn(tokens * max(1, top_k) + 2, hidden).to(C.BF16)
    places = weights = None
    if top_k:
        places = torch.randperm(tokens * top_k, generator=g, device=DEV).to(torch.int32).view(tokens, top_k)
        places[::3, -1] = -1
        weights = torch.rand(tokens, top_k, generator=g, device=DEV)
    post = 1 + 0.1 * randn(hidden) if variant & 1 else None
    pre = 1 + 0.1 * randn(hidden) if variant < 3 else None
    gate = GATES[variant]
    gate = {"none": None, "channel": randn(hidden), "token": randn(tokens, 1), "full": randn(tokens, hidden)}[gate]
    gate = None if gate is None else gate.to(C.BF16)
    scale = [1.0, 0.3, -2.0, 1.0][variant]
    out = None if pre is None else torch.zeros_like(h)
    h_out = h.clone() if variant == 2 else torch.zeros_like(h)
    serve.block_norm(L, h_out if variant == 2 else h, x, h_out, out=out, places=places, weights=weights, post=post, gate=gate,
                     scale=scale, pre=pre)
    within(h_out, *C.block(h, x, places, weights, post, gate, scale))
    if pre is not None:
        within(out, *C.norm(h_out, pre))
    assert L.device_error() == 0


def test_block_edges(L):
    """The norm of h alone; rows without any place; a zero row; strides; a bad place is left out (code 14); NaN stays in its row."""
    from paia_gemv import serve
    g = gen(21)
    big = torch.randn(12, 3 * 64, generator=g, device=DEV).to(C.BF16)
    h = big[:, 64:128]
    pre = 1 + 0.1 * torch.randn(64, generator=g, device=DEV)
    out = torch.zeros(12, 64, dtype=C.BF16, device=DEV)
    assert serve.block_norm(L, h, out=out, pre=pre) is out
    within(out, *C.norm(h, pre))
    x = torch.randn(20, 64, generator=g, device=DEV).to(C.BF16)
    x[4], x[9, 3] = 0, float("nan")
    places = torch.randint(0, 9, (12, 4), generator=g, device=DEV).to(torch.int32)
    places[2], places[3], places[5, 1] = -1, 4, 9
    weights = torch.rand(12, 4, generator=g, device=DEV)
    to = torch.full((12, 128), 7.0, dtype=C.BF16, device=DEV)
    serve.block_norm(L, h, x, to[:, :64], out=out, places=places, weights=weights, post=pre, pre=pre)
    ok = [i for i in range(12) if i != 5]
    want, bound = C.block(h[ok], x, places[ok], weights[ok], pre)
    within(to[ok, :64], want, bound)
    assert torch.equal(to[2, :64], h[2]) and torch.equal(to[3, :64], h[3]) and bool((to[:, 64:] == 7.0).all())
    assert torch.isnan(to[5, :64].float()).all() and torch.isnan(out[5].float()).all()
    places[5, 1], places[6, 0] = 20, -2
    serve.block_norm(L, h, x, to[:, :64], places=places, weights=weights)
    torch.cuda.synchronize()
    assert L.device_error() == 14 and L.device_error() == 0
    places[5, 1], places[6, 0] = -1, -1
    within(to[:, :64], *C.block(h, x, places, weights))
    serve.block_norm(L, torch.zeros(0, 64, dtype=C.BF16, device=DEV), out=torch.zeros(0, 64, dtype=C.BF16, device=DEV), pre=pre)


def test_a_block_of_experts(L, ws):
    """The operators one after another as a layer runs them, captured once and replayed on new inputs."""
    from paia_gemv import serve
    g, t, e, k, hid, inter = gen(31), 37, 12, 3, 256, 192
    gu, gus, gu_v = C.weights(e, 2 * inter, hid, "fp8", g, DEV)
    dn, dns, dn_v = C.weights(e, hid, inter, "bf16", g, DEV)
    pre = 1 + 0.1 * torch.randn(hid, generator=g, device=DEV)
    h, a, logits = (torch.zeros(t, n, dtype=C.BF16, device=DEV) for n in (hid, hid, e))
    mid, y = torch.zeros(t * k, inter, dtype=C.BF16, device=DEV), torch.zeros(t * k, hid, dtype=C.BF16, device=DEV)
    h_out, out = torch.zeros_like(h), torch.zeros_like(h)
    pos = torch.arange(t, device=DEV, dtype=torch.int32)
    r = serve.routing(L, t, e, k)

    def layer():
        serve.block_norm(L, h, out=a, pre=pre)
        serve.route(L, logits, r, positions=pos)
        serve.expert_matmul(L, gu, a, r.offsets, mid, ws, scales=gus, rows=r.rows, silu=True)
        serve.expert_matmul(L, dn, mid, r.offsets, y, ws)
        serve.block_norm(L, h, y, h_out, out=out, places=r.places, weights=r.weights, pre=pre)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for seed in range(3):
        q = gen(seed)
        h.copy_(torch.randn(t, hid, generator=q, device=DEV))
        logits.copy_(torch.randn(t, e, generator=q, device=DEV))
        pos[seed] = -1
        graph.replay()
        torch.cuda.synchronize()
        n = int(r.offsets[-1])
        assert n == (t - seed - 1) * k
        within(a, *C.norm(h, pre))
        within(mid[:n], *C.matmul(gu_v, a, r.offsets, r.rows, True, split=True))
        within(y[:n], *C.matmul(dn_v, mid, r.offsets))
        within(h_out, *C.block(h, y, r.places, r.weights))
        within(out, *C.norm(h_out, pre))
    assert L.device_error() == 0
