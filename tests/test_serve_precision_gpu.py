"""How exactly the serving operators compute what they keep in fewer than 32 bits, at inputs that show it: probabilities and
queries of an e4m3 cache's attention (f16 next to the stored bytes), and the bytes that an e4m3 cache stores."""
import math

import pytest
import torch

import serve_cases as C
from serve_cases import BF16, E4M3, F32, HALF

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paia_gemv import load_lib
    lib = load_lib()
    lib.device_error(True)
    return lib


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol, what=""):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs() - tol
    assert not off.numel() or off.max().item() <= 0, (what, off.max().item(), tol.flatten()[off.argmax()].item())


def attention8(q, k, v, table, lens, scale):
    """(out, lse, bound of out, bound of lse) of an e4m3 cache without scales, as serve_cases.attention, but with what f16
    may lose told apart by size: a probability is rounded by 2^-11 of its value down to 2^-29 of the largest and is off by
    2^-40 of that below (f16's half step of 2^-25 under 2^15), a query element exact (8 bits) down to 2^-32 of its head's
    largest and off by 2^-40 of that below."""
    f = torch.float64
    b, h, hd = q.shape
    kv, page = k.shape[2], k.shape[1]
    out, lse = torch.zeros(b, h, hd, dtype=f, device=q.device), torch.zeros(b, h, dtype=f, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lens):
        pos = torch.arange(n, device=q.device)
        rows = table[i].long()[pos // page]
        kk, vv = k[rows, pos % page].to(f), v[rows, pos % page].to(f)
        for j in range(kv):
            hs = slice(j * (h // kv), (j + 1) * (h // kv))
            qq = q[i, hs].to(f)
            s = scale * (qq @ kk[:, j].T)
            ds = scale * (hd + 16) * F32 * (qq.abs() @ kk[:, j].abs().T) + 4 * F32 * s.abs()
            ds = ds + scale * 2.0 ** -40 * qq.abs().amax(-1, keepdim=True) * kk[:, j].abs().sum(-1)
            p = torch.softmax(s, -1)
            z = torch.logsumexp(s, -1)
            # an exponent's error moves its own term and the sum that it is divided by: ds of the term, and of the sum the
            # terms' ds by their weight
            e = ds + (p * ds).sum(-1, keepdim=True) + 2.0 ** -20 + (n / 16 + 64) * 2 * F32
            e = e + 2 * F32 * (s.amax(-1, keepdim=True) - s + 16)            # the difference that ex2 is taken of
            pe = p * 2.0 ** -11 + 2.0 ** -40 * torch.exp(s.amax(-1) - z)[:, None]
            out[i, hs] = p @ vv[:, j]
            tol[i, hs] = ((p * e + pe) @ vv[:, j].abs()) * (1 + 2.0 ** -7) + HALF[BF16] * out[i, hs].abs() + 1e-38
            lse[i, hs] = z
            tol_lse[i, hs] = ((p * ds).sum(-1) + 2.0 ** -20 + (n / 16 + 64) * F32
                              + 4 * F32 * (z.abs() + s.abs().amax(-1) + 16))
    return out, lse, tol, tol_lse


def call(L, q, k, v, table, lens, scale):
    from paia_gemv import serve
    b, h, hd = q.shape
    out, lse = torch.empty_like(q), torch.empty(b, h, device="cuda")
    serve.paged_attention(L, q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out,
                          serve.attention_workspace(L, h, k.shape[2], hd), scale=scale, lse=lse)
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    want = attention8(q, k, v, table, lens, scale)
    within(out, want[0], want[2], "out")
    within(lse, want[1], want[3], "lse")


SHAPES = [(8, 2, 128), (4, 2, 64), (6, 1, 96), (4, 2, 256), (32, 2, 128), (12, 1, 64), (16, 1, 256)]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("gap", [0, 8, 14, 16, 18, 19.5])
def test_e4m3_small_probabilities_beside_a_large_one(L, heads, kv, hd, gap):
    """One position whose score lies `gap` above the others' middle and whose v is 0, at the front, in the middle and at the
    end: the output is what the small probabilities leave."""
    lens = [4000, 3001, 2500, 300, 40]
    g = gen(21)
    k, v, table = C.paged(lens, kv, hd, 16, E4M3, "cuda", g)
    scale = max(gap, 1) / 2048.0
    q = torch.randn(len(lens), heads, hd, generator=g, device="cuda")
    q = (q / (scale * 30 * math.sqrt(hd))).to(BF16)               # the other scores: N(0, 1)
    q[:, :, 0] = 8.0
    k[..., 0] = 0.0
    for b, at in enumerate((0, 1500, 2499, 150, 39)):
        pg = table[b, at // 16].item()
        k[pg, at % 16] = 0.0
        k[pg, at % 16, :, 0] = 256.0 if gap else 0.0              # score 8 * 256 * scale = gap
        v[pg, at % 16] = 0.0
    call(L, q, k, v, table, lens, scale)


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("small", [0, 10, 16, 20, 24])
def test_e4m3_small_query_elements_beside_a_large_one(L, heads, kv, hd, small):
    """A query whose largest element meets zeros in every key: the scores come from elements 2^-small times as large."""
    lens = [2100, 500, 33]
    g = gen(22)
    k, v, table = C.paged(lens, kv, hd, 16, E4M3, "cuda", g)
    q = (torch.randn(len(lens), heads, hd, generator=g, device="cuda") * 2.0 ** -small).to(BF16)
    q[:, :, 0] = 5.0
    k[..., 0] = 0.0
    call(L, q, k, v, table, lens, 2.0 ** small / 30 / math.sqrt(hd))


@pytest.mark.parametrize("size", [-120, -60, -20, 40, 100])
def test_e4m3_queries_of_any_size(L, size):
    """Scores of ordinary size from queries that f16 could not hold, and scale to match."""
    lens = [700, 40]
    g = gen(23)
    k, v, table = C.paged(lens, 2, 128, 16, E4M3, "cuda", g)
    q = (torch.randn(2, 8, 128, generator=g, device="cuda") * 2.0 ** size).to(BF16)
    call(L, q, k, v, table, lens, 2.0 ** -size / 30 / math.sqrt(128))


# ------------------------------------------------------------------ what an e4m3 cache stores

def nearest8(x):
    """The e4m3 value nearest to x (ties to even, at most 448), and how far x is from the next border between two of them."""
    a = x.abs().clamp(max=448.0)
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (e - 4).clamp(min=-9))
    r = a / step
    far = torch.where(x.abs() >= 448, torch.full_like(a, math.inf), ((r - torch.floor(r)) - 0.5).abs() * step)
    return torch.sign(x) * torch.round(r) * step, far


def same_bytes(pool, want, unsure=None):
    """The stored values (pool [..., hd]) are the nearest ones, but where the exact value is too near a border to tell."""
    value, far = nearest8(want)
    sure = torch.ones_like(far, dtype=torch.bool) if unsure is None else far > unsure
    assert sure.double().mean().item() > 0.99
    bad = (pool.double() != value) & sure
    assert not bad.any(), (int(bad.sum()), pool.double()[bad][:4].tolist(), want[bad][:4].tolist())
    return int((far < 1e-5 * value.abs()).sum())


def borders(g):
    """(l, scale) pairs whose quotient lies on a border between two e4m3 values or a few fp32 steps beside it: every bf16
    mantissa against every border of a binade and every subnormal one."""
    l = 1 + torch.arange(128, dtype=torch.float64) / 128
    normal = (2 * torch.arange(8, 16, dtype=torch.float64) + 1) / 16
    m = torch.cat([normal, normal * 2.0 ** -6, normal * 2.0 ** 7, (2 * torch.arange(8, dtype=torch.float64) + 1) * 2.0 ** -10])
    s = (l[:, None] / m).float()
    s = s[..., None].view(torch.int32) + torch.arange(-3, 4, dtype=torch.int32)
    s, two = s.view(torch.float32), torch.exp2(torch.randint(-9, 9, s.shape, generator=g).double())
    return (l[:, None, None] * two).reshape(-1), (s * two.float()).reshape(-1)


def test_e4m3_rows_at_borders(L):
    """Keys and values that are not turned (position 0, no norm), exactly on the borders and beside them."""
    from paia_gemv import serve
    l, s = borders(torch.Generator().manual_seed(3))
    kv, hd = len(l), 16
    sign = torch.where(torch.arange(hd) % 3 == 1, -1.0, 1.0).double()
    rows = (l[:, None] * sign).to(BF16)
    assert torch.equal(rows.double(), l[:, None] * sign)
    qkv = torch.cat([torch.zeros(hd, dtype=BF16), rows.reshape(-1), rows.reshape(-1)])[None].cuda()
    k = torch.zeros(1, 1, kv, hd, dtype=E4M3, device="cuda")
    v = torch.zeros_like(k)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    sc = s.cuda()
    serve.qkv_rope_cache(L, qkv, zero, serve.rope_inv_freq(16, 1e4), torch.empty(1, 1, hd, dtype=BF16, device="cuda"), k, v,
                         zero.view(1, 1), k_scale=sc, v_scale=sc)
    want = (rows.double() / s.double()[:, None]).cuda()
    assert same_bytes(v[0, 0], want) > 0 and same_bytes(k[0, 0], want) > 0
    assert L.device_error(True) == 0


@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 32), (96, 96), (256, 256), (80, 16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_e4m3_rows_are_the_nearest_values(L, hd, rot, inter, norm):
    """Turned and normed keys, and values, of many tokens; then of one token whose scales put an element of every key head
    on a border or a few fp32 steps beside it."""
    from paia_gemv import serve
    g = gen(31)
    eps = 2.0 ** -17
    freq = serve.rope_inv_freq(rot, 10000.0)
    kn = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if norm else None

    def run(qkv, pos, kv, ks, vs):
        n = len(pos)
        k = torch.zeros(n, 1, kv, hd, dtype=E4M3, device="cuda")
        v = torch.zeros_like(k)
        table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].expand(n, int(pos.max()) + 1).contiguous()
        serve.qkv_rope_cache(L, qkv, pos, freq, torch.empty(n, 1, hd, dtype=BF16, device="cuda"), k, v, table, k_norm=kn,
                             eps=eps, interleaved=inter, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        assert L.device_error(True) == 0
        return k[:, 0], v[:, 0]

    def exact(qkv, pos, kv):
        (_, wk, wv), (_, mk, _) = C.rope(qkv, pos, freq, 1, kv, hd, None, kn, eps, inter)
        # fp64: some steps of 2^-53 of the pair, and the angle's own step
        return wk, wv, mk * (2.0 ** -46 + pos.double().abs()[:, None, None] * 2.0 ** -50)

    kv, n = 3, 400
    qkv = (3 * torch.randn(n, (1 + 2 * kv) * hd, generator=g, device="cuda")).to(BF16)
    pos = torch.randint(0, 900, (n,), generator=g, device="cuda", dtype=torch.int32)
    ks, vs = (1 + 0.2 * torch.rand(2, kv, generator=g, device="cuda")) / 20
    k, v = run(qkv, pos, kv, ks, vs)
    wk, wv, ek = exact(qkv, pos, kv)
    same_bytes(k, wk / ks.double()[:, None], ek / ks.double()[:, None])
    same_bytes(v, wv / vs.double()[:, None])

    kv = 4096
    qkv = (3 * torch.randn(1, (1 + 2 * kv) * hd, generator=g, device="cuda")).to(BF16)
    pos = torch.tensor([777], dtype=torch.int32, device="cuda")
    wk, wv, ek = exact(qkv, pos, kv)
    at = torch.randint(0, hd, (kv,), generator=g, device="cuda")
    border = (2 * torch.randint(8, 16, (kv,), generator=g, device="cuda").double() + 1) / 16
    scales = []
    for w in (wk[0], wv[0]):
        x = w[torch.arange(kv, device="cuda"), at].abs().clamp(min=2.0 ** -10)
        step = torch.randint(-4, 5, (kv,), generator=g, device="cuda", dtype=torch.int32)
        scales.append(((x / border).float().view(torch.int32) + step).view(torch.float32))
    ks, vs = scales
    k, v = run(qkv, pos, kv, ks, vs)
    hit = same_bytes(k[0], wk[0] / ks.double()[:, None], ek[0] / ks.double()[:, None])
    assert same_bytes(v[0], wv[0] / vs.double()[:, None]) > kv // 2 and hit > kv // 2
