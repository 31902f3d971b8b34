"""The serving operators at the edges of what they take: errors beside one another, batches beyond the size that one scan
finds its place in, infinities and NaN."""

import math

import pytest
import torch

import serve_cases as C
from serve_cases import BF16, E4M3

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paia_gemv import load_lib
    lib = load_lib()
    while lib.device_error(True) > 0:
        pass
    return lib


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_errors_of_two_operators_are_both_reported(L):
    """A bad page id, a bad position and a bad adapter id between two reads: each is returned once."""
    from paia_gemv import serve
    z = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda")   # noqa: E731
    serve.paged_attention(L, z(1, 2, 64), z(2, 16, 1, 64), z(2, 16, 1, 64), i32([[7]]), i32([16]), z(1, 2, 64),
                          serve.attention_workspace(L, 2, 1, 64))
    serve.qkv_rope_cache(L, z(1, 4 * 64), i32([-2]), serve.rope_inv_freq(64, 1e4), z(1, 2, 64), z(2, 16, 1, 64),
                         z(2, 16, 1, 64), i32([[0]]))
    serve.lora(L, z(1, 64), z(1, 8, 64), z(1, 64, 8), i32([5]), z(1, 64))
    torch.cuda.synchronize()
    assert [L.device_error(False), L.device_error(False)] == [10, 10]
    assert [L.device_error(True) for _ in range(4)] == [10, 12, 13, 0]


# ------------------------------------------------------------------ batches beyond one scan

@pytest.mark.parametrize("n,heads,kv,hd,dtype", [(1025, 4, 2, 64, BF16), (1100, 8, 1, 128, E4M3), (2100, 2, 2, 64, BF16),
                                                 (1057, 16, 1, 64, E4M3), (3300, 1, 1, 64, BF16)])
def test_attention_of_more_than_1024_sequences(L, n, heads, kv, hd, dtype):
    """A CTA finds the start of its run in two scans or more: empty, single-token and long sequences mixed, long ones at
    the borders of the lanes' shares."""
    from paia_gemv import serve
    share = (n + 31) // 32
    lens = [0 if b % 5 == 0 else 1 if b % 5 == 1 else (b * b) % 90 for b in range(n)]
    for b in (0, share - 1, share, 32 * (share // 32), n - 1, n // 2):
        lens[b] = 700 + b % 50
    g = gen(n)
    k, v, table = C.paged(lens, kv, hd, 16, dtype, "cuda", g)
    q = torch.randn(n, heads, hd, generator=g, device="cuda").to(BF16)
    out, lse = torch.full_like(q, 7.0), torch.full((n, heads), 7.0, device="cuda")
    sc = 1.0 if dtype is BF16 else 1 / 30
    serve.paged_attention(L, q, k, v, table, i32(lens), out, serve.attention_workspace(L, heads, kv, hd),
                          scale=sc / math.sqrt(hd), lse=lse)
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    want, wl, tol, tl = C.attention(q, k, v, table, lens, sc / math.sqrt(hd))
    live = torch.tensor([x > 0 for x in lens], device="cuda")
    assert torch.isfinite(out).all() and torch.isfinite(lse[live]).all()
    assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - wl).abs()[live] <= tl[live]).all()
    assert (out[~live] == 0).all() and (lse[~live] == -math.inf).all()


@pytest.mark.parametrize("n", [1, 40, 700])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_attention_without_pages(L, n, dtype):
    """A page table of no columns: every sequence is empty, and a length above 0 is cut to that (code 11)."""
    from paia_gemv import serve
    pool = torch.full((1, 16, 2, 64), math.nan, device="cuda").to(dtype)
    q = torch.ones(n, 8, 64, dtype=BF16, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full((n, 8), 7.0, device="cuda")
    ws = serve.attention_workspace(L, 8, 2, 64)
    for lens, code in ((i32([0] * n), 0), (i32([0] * (n - 1) + [5]), 11)):
        serve.paged_attention(L, q, pool, pool, torch.empty(n, 0, dtype=torch.int32, device="cuda"), lens, out.fill_(7), ws, lse=lse)
        torch.cuda.synchronize()
        assert L.device_error(True) == code and (out == 0).all() and (lse == -math.inf).all()


# ------------------------------------------------------------------ infinities and NaN

SPLITS = [[17], [40, 3000], [3] * 200]                           # a cluster per unit, the list, CTAs of two warps


def attend(L, q, k, v, table, lens, scale=None):
    from paia_gemv import serve
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    serve.paged_attention(L, q, k, v, table, i32(lens), out, serve.attention_workspace(L, q.shape[1], k.shape[2], q.shape[2]),
                          scale=scale, lse=lse)
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    return out, lse


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64), (16, 1, 128), (4, 2, 256), (12, 1, 96)])
@pytest.mark.parametrize("lens", SPLITS)
def test_attention_infinite_scores(L, heads, kv, hd, lens):
    """bf16 keys of -inf along a query's positive element: those positions have no weight, and a head whose scores are all
    -inf gets zeros and -inf, whatever lies in the other sequences; +inf makes its kv head's outputs NaN."""
    g = gen(7)
    k, v, table = C.paged(lens, kv, hd, 16, BF16, "cuda", g)
    q = torch.randn(len(lens), heads, hd, generator=g, device="cuda").to(BF16)
    q[..., 0] = 1.0
    n, last = lens[0], kv - 1
    rows = table[0].long()[torch.arange(n, device="cuda") // 16], torch.arange(n, device="cuda") % 16
    hit = slice(heads - heads // kv, heads)
    clean, clean_lse = attend(L, q, k, v, table, lens)

    def others(out, lse):
        """Everything but sequence 0's last kv head is as it was."""
        out, lse = out.clone(), lse.clone()
        out[0, hit], lse[0, hit] = clean[0, hit], clean_lse[0, hit]
        return torch.equal(out, clean) and torch.equal(lse, clean_lse)

    keep = k[rows[0], rows[1], last, 0].clone()
    some = torch.arange(n, device="cuda") % 3 == 1               # every third position at -inf
    k[rows[0][some], rows[1][some], last, 0] = -math.inf
    out, lse = attend(L, q, k, v, table, lens)
    kk, vv = (x[rows[0], rows[1], last].double() for x in (k, v))
    want = torch.softmax(torch.einsum("hd,nd->hn", q[0, hit].double(), kk) * hd ** -0.5, -1) @ vv
    # scores of N(0, 1) rows: fp32 sums of head_dim products are off by at most hd^-0.5 (hd + 16) 2^-23 sum |q k|, which is
    # 3.5e-4 at 256 (sum |q k| is 0.64 hd); a probability and the sum it is divided by move by twice that, P is two bf16
    # (2^-16), and sum p |v| is below 2: 2e-3; the output's half step
    assert others(out, lse) and ((out[0, hit].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2e-3).all()
    k[rows[0], rows[1], last, 0] = -math.inf
    out, lse = attend(L, q, k, v, table, lens)
    assert others(out, lse) and (out[0, hit] == 0).all() and (lse[0, hit] == -math.inf).all()
    k[rows[0], rows[1], last, 0] = keep
    k[rows[0][-1], rows[1][-1], last, 0] = math.inf
    out, lse = attend(L, q, k, v, table, lens)
    assert others(out, lse) and out[0, hit].isnan().all() and not lse[0, hit].isfinite().any()


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64), (16, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("lens", SPLITS)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_attention_infinite_values(L, heads, kv, hd, lens, value):
    """An infinity or a NaN in v makes its dimension NaN or infinite, and nothing else changes."""
    g = gen(8)
    k, v, table = C.paged(lens, kv, hd, 16, BF16, "cuda", g)
    q = torch.randn(len(lens), heads, hd, generator=g, device="cuda").to(BF16)
    clean, clean_lse = attend(L, q, k, v, table, lens)
    at = lens[0] - 1
    v[table[0, at // 16], at % 16, kv - 1, 5] = value
    out, lse = attend(L, q, k, v, table, lens)
    hit = slice(heads - heads // kv, heads)
    assert not out[0, hit, 5].isfinite().any()
    out[0, hit, 5] = clean[0, hit, 5]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_rope_infinities_and_nan(L, dtype, value):
    """An infinity or a NaN in a head's row reaches what the formulas say it reaches: of a head that is only turned its pair,
    of a normed one every element, of v itself alone; an e4m3 cache keeps NaN and stores infinities as 448."""
    from paia_gemv import serve
    g = gen(12)
    hd, at = 64, 5
    freq = serve.rope_inv_freq(hd, 1e4)
    kn = torch.ones(hd, device="cuda")

    def run(qkv, norm):
        q = torch.empty(3, 2, hd, dtype=BF16, device="cuda")
        k = torch.zeros(3, 16, 1, hd, dtype=dtype, device="cuda")
        v = torch.zeros_like(k)
        ko = torch.empty(3, 1, hd, dtype=BF16, device="cuda")
        serve.qkv_rope_cache(L, qkv, i32([3, 9, 4]), freq, q, k, v, i32([[0], [1], [2]]), k_norm=kn if norm else None, k_out=ko)
        torch.cuda.synchronize()
        assert L.device_error(True) == 0
        row = torch.arange(3, device="cuda"), torch.tensor([3, 9, 4], device="cuda")
        return q, k[row].float(), v[row].float(), ko
    qkv = torch.randn(3, 4 * hd, generator=g, device="cuda").to(BF16)
    for norm in (False, True):
        q0, k0, v0, ko0 = run(qkv, norm)
        bad = qkv.clone()
        bad[1, at] = bad[1, 2 * hd + at] = bad[1, 3 * hd + at] = value        # q's head 0, k, v
        q, k, v, ko = run(bad, norm)
        pair = [at, at + hd // 2]
        assert not q[1, 0, pair].isfinite().any()
        q[1, 0, pair] = q0[1, 0, pair]
        assert torch.equal(q, q0)
        got = k[1, 0, pair]
        # turned: infinite or NaN; normed: x / sqrt(inf) is NaN for the infinity, 0 for finite ones, NaN all for NaN
        assert not ko[1, 0, pair].isfinite().any()
        assert (got.isnan() | (got.abs() == (math.inf if dtype is BF16 else 448))).all()
        rest = [i for i in range(hd) if i not in pair]
        if norm:
            assert (k[1, 0, rest].isnan().all() if math.isnan(value) else (k[1, 0, rest] == 0).all())
        else:
            assert torch.equal(k[1, 0, rest], k0[1, 0, rest])
        assert torch.equal(k[[0, 2]], k0[[0, 2]]) and torch.equal(ko[[0, 2]], ko0[[0, 2]])
        want = torch.tensor(value, device="cuda") if dtype is BF16 or math.isnan(value) else torch.tensor(math.copysign(448.0, value), device="cuda")
        assert v[1, 0, at].isnan() if math.isnan(value) else v[1, 0, at] == want
        v[1, 0, at] = v0[1, 0, at]
        assert torch.equal(v, v0)


@pytest.mark.parametrize("M", [3, 12, 300])
@pytest.mark.parametrize("rank", [8, 40, 72])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_lora_infinities_and_nan(L, M, rank, value):
    """An infinity or a NaN in x reaches its row, in A the rows of its adapter, in B their column, in base its element;
    nothing else changes."""
    from paia_gemv import serve
    g = gen(14)
    K, N, bank = 264, 136, 3
    x = torch.randn(M, K, generator=g, device="cuda").to(BF16)
    a = (torch.randn(bank, rank, K, generator=g, device="cuda") / 16).to(BF16)
    b = torch.randn(bank, N, rank, generator=g, device="cuda").to(BF16)
    base = torch.randn(M, N, generator=g, device="cuda").to(BF16)
    ad = i32([m % 4 - 1 for m in range(M)])

    def run(x=x, a=a, b=b, base=base):
        out = torch.full((M, N), 7.0, dtype=BF16, device="cuda")
        serve.lora(L, x, a, b, ad, out, base=base)
        torch.cuda.synchronize()
        assert L.device_error(True) == 0
        return out

    def bad(t, *at):
        t = t.clone()
        t[at] = value
        return t
    clean = run()
    mine = ad == 0                                               # rows 1, 5, 9, ... have adapter 0
    full = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    hit = full.clone()
    hit[1] = True
    col = full.clone()
    col[mine, 77] = True
    one = full.clone()
    one[1, 9] = True
    for out, where in ((run(x=bad(x, 1, 200)), hit), (run(a=bad(a, 0, rank - 1, 3)), mine[:, None].expand(M, N)),
                       (run(b=bad(b, 0, 77, rank - 1)), col), (run(base=bad(base, 1, 9)), one)):
        assert not out[where].isfinite().any() and torch.equal(out[~where], clean[~where])
    assert torch.equal(run(x=bad(x, 0, 200)), clean)             # a row without an adapter: its x is not used


# ------------------------------------------------------------------ a row among others

@pytest.mark.parametrize("rank,ranks", [(16, None), (72, [72, 5, 40, 16])])
def test_lora_row_among_any_others(L, rank, ranks):
    """A row gives the same result, within the sums' rounding, alone and among rows of its own and other adapters (the
    division of K and the order of the sums follow the call), and the same bits whenever a call is repeated."""
    from paia_gemv import serve
    g = gen(15)
    K, N, bank = 1032, 264, 4
    a = (torch.randn(bank, rank, K, generator=g, device="cuda") / math.sqrt(K)).to(BF16)
    b = (torch.randn(bank, N, rank, generator=g, device="cuda") * 0.1).to(BF16)
    x = torch.randn(600, K, generator=g, device="cuda").to(BF16)
    base = torch.randn(600, N, generator=g, device="cuda").to(BF16)
    x[:], base[:] = torch.where(torch.arange(600, device="cuda")[:, None] % 7 == 0, x[:1], x), \
        torch.where(torch.arange(600, device="cuda")[:, None] % 7 == 0, base[:1], base)
    rk = None if ranks is None else i32(ranks)
    rows = []
    for M, other in ((1, 0), (8, 0), (9, 0), (40, 0), (40, 1), (300, 2), (600, 1)):
        ad = i32([2 if m % 7 == 0 else (2 if other == 0 else (m * other) % (bank + 1) - 1) for m in range(M)])
        out, again = torch.empty(M, N, dtype=BF16, device="cuda"), torch.empty(M, N, dtype=BF16, device="cuda")
        for y in (out, again):
            serve.lora(L, x[:M], a, b, ad, y, base=base[:M], ranks=rk)
        want, tol = C.lora(x[:M], a, b, ad, base[:M], None, ranks)
        assert torch.equal(out, again) and ((out.double() - want).abs() <= tol).all()
        rows.append(out[::7])
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    want, tol = C.lora(x[:1], a, b, i32([2]), base[:1], None, ranks)
    for r in rows:
        assert ((r.double() - rows[0].double()).abs() <= 2 * tol).all()
