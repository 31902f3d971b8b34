"""The serving operators (paia_gemv.serve) on the GPU against their 64-bit plain forms, element by element within bounds
that follow from the number formats (serve_cases): paged attention over every head layout, page size, length and mask
that has its own path; norm + rotary + cache write; multi-request adapters; and the run of them that a decode step makes."""
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


@pytest.fixture(params=["extension", "ctypes"])
def route(request, monkeypatch):
    """Both ways a call takes: the extension's checks in C, and Python's."""
    from paia_gemv import serve
    if request.param == "ctypes":
        monkeypatch.setattr(serve, "_bind", None)
    else:
        assert serve._bind is not None, "csrc/serve_bind.cpp is not built"
    return request.param


def test_both_routes_make_the_same_calls(L, monkeypatch, route):
    """Strides, optional arguments and dimensions of one, whichever way the call takes."""
    seen = []

    class Spy:
        def __getattr__(self, name):
            return getattr(serve_bind, name)

    from paia_gemv import serve
    serve_bind = serve._bind
    if route == "extension":
        for name in ("paged_attention", "qkv_rope_cache", "lora"):
            real = getattr(serve_bind, name)
            setattr(Spy, name, staticmethod(lambda *a, real=real: seen.append(real(*a)) or seen[-1]))
        monkeypatch.setattr(serve, "_bind", Spy())
    for lens, heads, kv in (([1], 1, 1), ([40, 0, 300], 6, 2)):
        for dtype in (BF16, E4M3):
            call, out, lse, want = attend(L, lens, heads, kv, 64, 16, dtype, hnd=True, window=50)
            check(out, lse, want, lens)
    test_attention_strided_and_scaled(L)
    rope_case(L, 1, 1, 1, 64, 64)
    rope_case(L, 20, 6, 2, 128, 64, E4M3, inter=True, hnd=True, k_out=True)
    rope_case(L, 20, 6, 2, 128, 64, norm=False, in_place=True)
    lora_case(L, 1, 64, 64, 8, 1, [0])
    lora_case(L, 20, 128, 72, 16, 3, [m % 4 - 1 for m in range(20)], ranks=[3, 16, 9], in_place=True)
    test_lora_strided(L)
    if route == "extension":
        assert seen and set(seen) == {0}                         # the extension made every call itself


def test_refusals_on_the_device(L, route):
    """What a call must not be given raises, whichever way it takes, and nothing is launched."""
    from paia_gemv import serve
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")   # noqa: E731
    i32 = torch.int32
    ws = serve.attention_workspace(L, 4, 2, 64)
    good = dict(q=z(3, 4, 64), k_pages=z(5, 16, 2, 64), v_pages=z(5, 16, 2, 64), page_table=z(3, 6, dtype=i32),
                lens=z(3, dtype=i32), out=torch.ones(3, 4, 64, dtype=BF16, device="cuda"), workspace=ws)
    for bad, err in ((dict(q=z(3, 4, 64).float()), ValueError), (dict(lens=torch.zeros(3, dtype=i32)), ValueError),
                     (dict(v_pages=z(4, 16, 2, 64)), ValueError), (dict(k_scale=z(2, dtype=torch.float32)), ValueError),
                     (dict(page_table=z(3, 6, dtype=torch.int64)), ValueError), (dict(lse=z(3, 4)), ValueError),
                     (dict(workspace=serve.attention_workspace(L, 4, 4, 64)), ValueError), (dict(window=-1), RuntimeError),
                     (dict(scale=0.0), RuntimeError), (dict(q=z(3, 4, 68)[:, :, :64]), RuntimeError),
                     (dict(out=z(3, 1, 64).expand(3, 4, 64)), RuntimeError)):
        with pytest.raises(err):
            serve.paged_attention(L, **dict(good, **bad))
    assert (good["out"] == 1).all()
    good = dict(qkv=z(3, 8 * 64), positions=z(3, dtype=i32), inv_freq=z(32, dtype=torch.float64), q_out=z(3, 4, 64),
                k_pages=z(5, 16, 2, 64), v_pages=z(5, 16, 2, 64), page_table=z(3, 6, dtype=i32))
    for bad, err in ((dict(qkv=z(3, 7 * 64)), ValueError), (dict(inv_freq=z(32, dtype=torch.float32)), ValueError),
                     (dict(page_table=z(2, 6, dtype=i32)), ValueError), (dict(seq=z(2, dtype=i32)), ValueError),
                     (dict(q_norm=z(64)), ValueError), (dict(inv_freq=z(40, dtype=torch.float64)), RuntimeError),
                     (dict(eps=-1.0), RuntimeError)):
        with pytest.raises(err):
            serve.qkv_rope_cache(L, **dict(good, **bad))
    good = dict(x=z(3, 64), a=z(2, 8, 64), b=z(2, 40, 8), adapter=z(3, dtype=i32), out=z(3, 40))
    for bad, err in ((dict(x=z(3, 32)), ValueError), (dict(b=z(2, 40, 16)), ValueError), (dict(base=z(2, 40)), ValueError),
                     (dict(adapter=z(3, dtype=torch.int64)), ValueError),
                     (dict(a=z(2, 12, 64), b=z(2, 40, 12)), RuntimeError),
                     (dict(out=z(1, 40).expand(3, 40)), RuntimeError)):
        with pytest.raises(err):
            serve.lora(L, **dict(good, **bad))
    torch.cuda.synchronize()
    assert L.device_error(True) == 0


# ------------------------------------------------------------------ attention

def attend(L, lens, heads, kv, hd, page, dtype=BF16, hnd=False, window=0, scale=None, seed=1, q=None, ws=None):
    from paia_gemv import serve
    g = gen(seed)
    k, v, table = C.paged(lens, kv, hd, page, dtype, "cuda", g, hnd)
    if q is None:
        q = torch.randn(len(lens), heads, hd, generator=g, device="cuda").to(BF16)
    ks = vs = None
    if dtype is E4M3:
        ks = (1 + 0.2 * torch.rand(kv, generator=g, device="cuda")) / 30
        vs = (1 + 0.2 * torch.rand(kv, generator=g, device="cuda")) / 30
    out = torch.full((len(lens), heads, hd), 7.0, dtype=BF16, device="cuda")
    lse = torch.full((len(lens), heads), 7.0, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = serve.attention_workspace(L, heads, kv, hd) if ws is None else ws
    call = lambda: serve.paged_attention(L, q, k, v, table, n, out, ws, scale=scale, window=window,   # noqa: E731
                                         k_scale=ks, v_scale=vs, lse=lse)
    call()
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    want = C.attention(q, k, v, table, lens, hd ** -0.5 if scale is None else scale, window, ks, vs)
    return call, out, lse, want


def check(out, lse, want, lens):
    o, s, to, ts = want
    within(out, o, to, "out")
    live = torch.tensor([n > 0 for n in lens], device="cuda")
    within(lse[live], s[live], ts[live], "lse")
    assert (lse[~live] == -math.inf).all() and (out[~live] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (28, 4), (16, 2), (9, 1), (32, 2), (40, 2)])
def test_attention_heads_and_types(L, dtype, hd, heads, kv):
    lens = [33, 0, 1, 700, 16, 15, 17, 129]
    call, out, lse, want = attend(L, lens, heads, kv, hd, 16, dtype)
    check(out, lse, want, lens)


@pytest.mark.parametrize("page", [1, 5, 8, 12, 16, 24, 64, 256])
@pytest.mark.parametrize("hnd", [False, True])
def test_attention_pages_and_layouts(L, page, hnd):
    lens = [3 * page + 1, page, 1, 301, 2 * page - 1]
    for dtype in (BF16, E4M3):
        call, out, lse, want = attend(L, lens, 8, 2, 128, page, dtype, hnd)
        check(out, lse, want, lens)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [2], [16384], [20011, 1, 0, 3], [5] * 700, [0, 1] * 300 + [900],
                                  list(range(0, 400))])
def test_attention_lengths(L, lens):
    """One sequence split over the whole GPU, batches of more sequences than a CTA has threads, empty ones between."""
    call, out, lse, want = attend(L, lens, 8, 2, 64, 16)
    check(out, lse, want, lens)


@pytest.mark.parametrize("n", [0, 1, 15, 16, 17, 40, 100, 255, 1000, 2048, 2049, 4096, 4100])
def test_attention_small_calls(L, n):
    """One or two sequences of few heads (a cluster of CTAs per unit) around the lengths where parts fall empty and where
    another division takes over."""
    for heads, kv, hd, dtype, lens in ((8, 2, 128, BF16, [n]), (7, 1, 64, E4M3, [n, 3]), (8, 8, 96, BF16, [5, n]),
                                       (4, 4, 128, E4M3, [n]), (16, 2, 256, BF16, [n]), (12, 2, 256, E4M3, [n, 1])):
        call, out, lse, want = attend(L, lens, heads, kv, hd, 16, dtype)
        check(out, lse, want, lens)
        first = out.clone()
        for _ in range(3):
            call()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


@pytest.mark.parametrize("batch", [9, 14, 17, 19, 33, 37, 38, 74, 75])
@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, BF16), (128, E4M3), (256, E4M3)])
def test_attention_cluster_sizes(L, batch, hd, dtype):
    """Clusters of 8, 4 and 2 CTAs per unit and none, for units from none to as many tiles as they take."""
    most = 500 if hd >= 128 else 1000
    lens = [(97 * i * i + 31 * i) % most if i % 7 else 0 for i in range(batch)]
    lens[-1] = most
    for heads in (5, 14, 20):                                     # one unit of 8 rows, one of 16, two of 16
        call, out, lse, want = attend(L, lens, heads, 1, hd, 16, dtype)
        check(out, lse, want, lens)
        first = out.clone()
        call()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


@pytest.mark.parametrize("heads,kv,hd,dtype", [(8, 2, 128, BF16), (4, 4, 64, E4M3), (16, 1, 128, BF16), (4, 2, 256, BF16)])
@pytest.mark.parametrize("lens", [[17], [40, 3000], [3] * 200])
def test_attention_nan_stays_nan(L, heads, kv, hd, dtype, lens):
    """A NaN query makes its own head NaN in every division of the work; a NaN key in a part of its own (the last of 17
    positions) makes its kv head's outputs NaN; nothing else changes."""
    from paia_gemv import serve
    g = gen(9)
    k, v, table = C.paged(lens, kv, hd, 16, dtype, "cuda", g)
    q = torch.randn(len(lens), heads, hd, generator=g, device="cuda").to(BF16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = serve.attention_workspace(L, heads, kv, hd)

    def run():
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        serve.paged_attention(L, q, k, v, table, n, out, ws, lse=lse)
        return out, lse
    clean, clean_lse = run()
    q[0, 1, 5] = math.nan
    out, lse = run()
    assert out[0, 1].isnan().all() and lse[0, 1].isnan()
    out[0, 1], lse[0, 1] = clean[0, 1], clean_lse[0, 1]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
    q[0, 1, 5] = 0.0
    clean, clean_lse = run()
    at = lens[0] - 1
    k.view(torch.uint8 if dtype is E4M3 else torch.int16)[table[0, at // 16], at % 16, kv - 1, 3] = \
        0x7F if dtype is E4M3 else 0x7FFF
    out, lse = run()
    hit = slice(heads - heads // kv, heads)
    assert out[0, hit].isnan().all() and lse[0, hit].isnan().all()
    out[0, hit], lse[0, hit] = clean[0, hit], clean_lse[0, hit]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 1024])
def test_attention_window(L, window):
    lens = [1, window, window + 1, 3000, 0, 777]
    for dtype in (BF16, E4M3):
        call, out, lse, want = attend(L, lens, 4, 2, 128, 16, dtype, window=window)
        check(out, lse, want, lens)


def test_attention_sharp_scores_and_far_maximum(L):
    """Scores up to some hundreds, with the largest at the front, in the middle and at the end."""
    from paia_gemv import serve
    g = gen(4)
    lens = [2000, 2000, 2000]
    k, v, table = C.paged(lens, 2, 128, 16, BF16, "cuda", g)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(BF16)
    for b, at in enumerate((0, 1003, 1999)):
        for j in range(2):
            k[table[b, at // 16].item(), at % 16, j] = 6 * q[b, 4 * j]
    ws = serve.attention_workspace(L, 8, 2, 128)
    out, lse = torch.empty(3, 8, 128, dtype=BF16, device="cuda"), torch.empty(3, 8, device="cuda")
    serve.paged_attention(L, q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, ws, lse=lse)
    check(out, lse, C.attention(q, k, v, table, lens, 128 ** -0.5), lens)


def test_attention_strided_and_scaled(L):
    """q inside a fused projection's rows, out inside a wider buffer, its neighbours left alone."""
    from paia_gemv import serve
    g = gen(9)
    lens = [40, 7, 200]
    k, v, table = C.paged(lens, 2, 128, 16, BF16, "cuda", g)
    qkv = torch.randn(3, 12 * 128, generator=g, device="cuda").to(BF16)
    q = qkv[:, :8 * 128].view(3, 8, 128)
    wide = torch.full((3, 9, 160), 3.0, dtype=BF16, device="cuda")
    out = wide[:, :8, :128]
    lse = torch.zeros(3, 16, device="cuda")[:, :8]
    ws = serve.attention_workspace(L, 8, 2, 128)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    serve.paged_attention(L, q, k, v, table, n, out, ws, scale=0.3, lse=lse)
    check(out, lse, C.attention(q, k, v, table, lens, 0.3), lens)
    assert (wide[:, 8] == 3).all() and (wide[:, :, 128:] == 3).all()


def test_attention_same_bits_and_shared_workspace(L):
    """The join gives the same bits on every run, and one workspace serves batches of other sizes in turn."""
    from paia_gemv import serve
    ws = serve.attention_workspace(L, 8, 2, 128)
    a = attend(L, [9000, 17, 0, 2500], 8, 2, 128, 16, ws=ws)
    first = a[1].clone()
    b = attend(L, [1, 40], 8, 2, 128, 16, ws=ws, seed=2)
    check(b[1], b[2], b[3], [1, 40])
    for _ in range(20):
        a[0]()
        b[0]()
    torch.cuda.synchronize()
    assert torch.equal(a[1], first)
    counters = ws.buffer[:2560].view(torch.int32)
    assert (counters == 0).all()


def test_attention_graph_with_growing_lengths_and_streams(L):
    """A captured call follows lens, and calls on two streams with a workspace each do not disturb each other."""
    from paia_gemv import serve
    g = gen(11)
    k, v, table = C.paged([600, 600], 2, 128, 16, BF16, "cuda", g)
    q = torch.randn(2, 8, 128, generator=g, device="cuda").to(BF16)
    n = torch.tensor([1, 500], dtype=torch.int32, device="cuda")
    outs, graphs = [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        out, lse = torch.empty(2, 8, 128, dtype=BF16, device="cuda"), torch.empty(2, 8, device="cuda")
        ws = serve.attention_workspace(L, 8, 2, 128)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            for _ in range(3):
                serve.paged_attention(L, q, k, v, table, n, out, ws, lse=lse)
        outs.append((out, lse, ws))
        graphs.append(gr)
    for step in range(3):
        n.copy_(torch.tensor([1 + 17 * step, 500 + step], dtype=torch.int32))
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(5):
                    gr.replay()
        torch.cuda.synchronize()
        lens = n.tolist()
        want = C.attention(q, k, v, table, lens, 128 ** -0.5)
        for out, lse, _ in outs:
            check(out, lse, want, lens)
    assert L.device_error(True) == 0


def test_attention_far_offsets(L):
    """Pages beyond 2^31 elements of the pool."""
    from paia_gemv import serve
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    page, kv, hd = 16, 8, 128
    pages = (5 << 30) // (page * kv * hd * 2)                    # 5 GB per pool: byte and element offsets over 2^31
    k = torch.zeros(pages, page, kv, hd, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(3)
    ids = [pages - 1, 0, pages - 2]
    for i in ids:
        k[i] = torch.randn(page, kv, hd, generator=g, device="cuda").to(BF16)
        v[i] = torch.randn(page, kv, hd, generator=g, device="cuda").to(BF16)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 8, hd, generator=g, device="cuda").to(BF16)
    out, lse = torch.empty(1, 8, hd, dtype=BF16, device="cuda"), torch.empty(1, 8, device="cuda")
    serve.paged_attention(L, q, k, v, table, torch.tensor([45], dtype=torch.int32, device="cuda"), out,
                          serve.attention_workspace(L, 8, kv, hd), lse=lse)
    check(out, lse, C.attention(q, k, v, table, [45], hd ** -0.5), [45])


def test_attention_bad_indices_are_reported(L):
    """A page id outside the pool is not followed (code 10), lengths are cut to the table (code 11)."""
    from paia_gemv import serve
    g = gen(5)
    k, v, table = C.paged([64, 64], 2, 64, 16, BF16, "cuda", g)
    table = table[:, :4].contiguous()
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(BF16)
    out, ws = torch.empty(2, 4, 64, dtype=BF16, device="cuda"), serve.attention_workspace(L, 4, 2, 64)
    lens = torch.tensor([64, 64], dtype=torch.int32, device="cuda")
    for bad in (-1, k.shape[0], 0x7FFFFFFF):
        t2 = table.clone()
        t2[1, 2] = bad
        serve.paged_attention(L, q, k, v, t2, lens, out, ws)
        assert L.device_error(True) == 10
        want = C.attention(q, k, v, table, [64, 64], 64 ** -0.5)
        within(out[0], want[0][0], want[2][0])                   # the other sequence is untouched
    for bad in (65, 0x7FFFFFFF):
        serve.paged_attention(L, q, k, v, table, torch.tensor([bad, 64], dtype=torch.int32, device="cuda"), out, ws)
        assert L.device_error(True) == 11
        within(out, want[0], want[2])
    serve.paged_attention(L, q, k, v, table, torch.tensor([-5, 64], dtype=torch.int32, device="cuda"), out, ws)
    assert L.device_error(True) == 11 and (out[0] == 0).all()
    assert L.device_error(True) == 0


# ------------------------------------------------------------------ norm, rotary positions, cache write

def rope_case(L, tokens, heads, kv, hd, rot, dtype=BF16, norm=True, inter=False, page=16, start=0, hnd=False, seed=1,
              k_out=False, in_place=False):
    from paia_gemv import serve
    g = gen(seed)
    pos = torch.tensor([-1 if t % 7 == 5 else start + 3 * t for t in range(tokens)], dtype=torch.int32, device="cuda")
    top = max(1, int(pos.max()) + 1)
    seq = torch.tensor([t % 3 for t in range(tokens)], dtype=torch.int32, device="cuda")
    cols = -(-top // page)
    used = sorted({(int(s), int(p) // page) for s, p in zip(seq, pos) if p >= 0})
    table = torch.full((3, cols), -1, dtype=torch.int32)
    for i, (s, c) in enumerate(used):
        table[s, c] = len(used) - 1 - i
    shape = (len(used) + 1, kv, page, hd) if hnd else (len(used) + 1, page, kv, hd)
    pools = [torch.full(shape, 5.0, device="cuda").to(dtype) for _ in range(2)]
    k, v = (x.transpose(1, 2) if hnd else x for x in pools)
    qkv = torch.randn(tokens, (heads + 2 * kv) * hd, generator=g, device="cuda").to(BF16)
    src = qkv.clone()
    qn = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if norm else None
    kn = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if norm else None
    ks = vs = None
    if dtype is E4M3:
        ks = (1 + 0.2 * torch.rand(kv, generator=g, device="cuda")) / 60
        vs = (1 + 0.2 * torch.rand(kv, generator=g, device="cuda")) / 60
    freq = serve.rope_inv_freq(rot, 10000.0)
    q = qkv[:, :heads * hd].view(tokens, heads, hd) if in_place else torch.full((tokens, heads, hd), 9.0, dtype=BF16,
                                                                                device="cuda")
    ko = torch.full((tokens, kv, hd), 9.0, dtype=BF16, device="cuda") if k_out else None
    serve.qkv_rope_cache(L, qkv, pos, freq, q, k, v, table.cuda(), seq=seq, q_norm=qn, k_norm=kn, eps=1e-5,
                         interleaved=inter, k_scale=ks, v_scale=vs, k_out=ko)
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    (wq, wk, wv), (mq, mk, mv) = C.rope(src, pos, freq, heads, kv, hd, qn, kn, 1e-5, inter)
    live = pos >= 0
    # fp32: the mean square (head_dim / 16 + 8 steps), sqrt, division, two products, sine and cosine (4 steps), rotation
    arith = (hd / 16 + 32) * F32
    within(q[live], wq[live], HALF[BF16] * wq[live].abs() + arith * 1.01 * mq[live] + 1e-38, "q")
    keep = src[:, :heads * hd].view(tokens, heads, hd) if in_place else torch.full_like(q, 9.0)
    assert torch.equal(q[~live], keep[~live])
    if k_out:
        within(ko[live], wk[live], HALF[BF16] * wk[live].abs() + arith * 1.01 * mk[live] + 1e-38, "k_out")
        assert (ko[~live] == 9).all()
    at = table.cuda()[seq[live].long(), (pos[live] // page).long()].long(), (pos[live] % page).long()
    for pool, want, mag, sc in ((k, wk, mk, ks), (v, wv, mv, vs)):
        got = pool[at].double()
        want, mag = want[live], mag[live]
        if sc is not None:
            want, mag = (want / sc.double()[:, None]).clamp(-448, 448), mag / sc.double()[:, None]
            # e4m3's step below 2^-6 is 2^-9
            tol = HALF[E4M3] * want.abs() + 2.0 ** -10 + 2.0 ** -40 * mag
        else:
            tol = HALF[BF16] * want.abs() + arith * 1.01 * mag + 1e-38
        within(got, want, tol, "cache")
        flat = pool.float().clone()
        flat[at] = 5.0
        assert (flat == 5.0).all()                               # every other row of the pools is as it was
    return q, k, v


@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 128), (96, 96), (256, 256), (128, 64), (80, 32), (16, 16), (64, 0),
                                    (256, 16)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_heads(L, hd, rot, inter):
    for dtype in (BF16, E4M3):
        rope_case(L, 13, 6, 2, hd, rot, dtype, inter=inter)


@pytest.mark.parametrize("tokens", [1, 2, 31, 400, 2500])
def test_rope_tokens(L, tokens):
    rope_case(L, tokens, 28, 4, 128, 128)
    rope_case(L, tokens, 3, 1, 64, 64, E4M3, hnd=True, norm=False)
    rope_case(L, tokens, 1, 1, 96, 48, hnd=True)


@pytest.mark.parametrize("start", [0, 130000, 1 << 22])
def test_rope_far_positions(L, start):
    rope_case(L, 20, 4, 2, 128, 128, start=start, page=4096)
    rope_case(L, 20, 4, 2, 128, 128, E4M3, start=start, page=4096)


def test_rope_in_place_and_key_output(L):
    rope_case(L, 40, 8, 2, 128, 128, in_place=True, k_out=True)
    rope_case(L, 40, 8, 2, 64, 32, in_place=True, k_out=True, inter=True, page=5)


def test_rope_without_cache(L):
    from paia_gemv import serve
    g = gen(2)
    qkv = torch.randn(9, 6 * 64, generator=g, device="cuda").to(BF16)
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    q, ko = torch.empty(9, 4, 64, dtype=BF16, device="cuda"), torch.empty(9, 1, 64, dtype=BF16, device="cuda")
    freq = serve.rope_inv_freq(64, 1e6)
    kn = torch.ones(64, device="cuda")
    serve.qkv_rope_cache(L, qkv, pos, freq, q, None, None, None, k_norm=kn, k_out=ko, kv_heads=1)
    (wq, wk, _), (mq, mk, _) = C.rope(qkv, pos, freq, 4, 1, 64, None, kn)
    within(q, wq, HALF[BF16] * wq.abs() + 64 * F32 * mq)
    within(ko, wk, HALF[BF16] * wk.abs() + 64 * F32 * mk)


def test_rope_saturates_e4m3(L):
    """Values beyond 448 scales are stored as 448, signs kept."""
    from paia_gemv import serve
    qkv = torch.full((1, 3 * 16), 1000.0, dtype=BF16, device="cuda")
    qkv[0, 16:32] *= -1
    k = torch.zeros(1, 1, 1, 16, dtype=E4M3, device="cuda")
    v = torch.zeros_like(k)
    q = torch.empty(1, 1, 16, dtype=BF16, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    serve.qkv_rope_cache(L, qkv, zero, serve.rope_inv_freq(16, 1e4), q, k, v, zero.view(1, 1))
    assert (k.float() == -448).all() and (v.float() == 448).all() and (q == 1000).all()


def test_rope_bad_indices_are_reported(L):
    """Bad pages (10), positions behind the table, sequences outside it and positions below -1 (12) store nothing."""
    from paia_gemv import serve
    g = gen(6)
    qkv = torch.randn(2, 4 * 64, generator=g, device="cuda").to(BF16)
    q = torch.empty(2, 2, 64, dtype=BF16, device="cuda")
    freq = serve.rope_inv_freq(64, 1e4)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    for pos, seq, table, code in (([3, 3], [0, 1], [[0], [-1]], 10), ([3, 3], [0, 1], [[0], [2]], 10),
                                  ([3, 16], [0, 1], [[0], [1]], 12), ([3, 3], [0, 2], [[0], [1]], 12),
                                  ([3, 3], [0, -1], [[0], [1]], 12), ([3, -2], [0, 1], [[0], [1]], 12)):
        k = torch.zeros(2, 16, 1, 64, dtype=BF16, device="cuda")
        v = torch.zeros_like(k)
        serve.qkv_rope_cache(L, qkv, i32(pos), freq, q, k, v, i32(table), seq=i32(seq))
        assert L.device_error(True) == code
        assert (k[1] == 0).all() and (v[1] == 0).all() and torch.equal(v[0, 3, 0], qkv[0, 3 * 64:])


# ------------------------------------------------------------------ adapters

def lora_case(L, M, K, N, rank, bank, adapter, ranks=None, base=True, scaling=True, in_place=False, seed=1, junk=False):
    from paia_gemv import serve
    g = gen(seed)
    x = torch.randn(M, K, generator=g, device="cuda").to(BF16)
    a = (torch.randn(bank, rank, K, generator=g, device="cuda") / math.sqrt(K)).to(BF16)
    b = (torch.randn(bank, N, rank, generator=g, device="cuda") * 0.1).to(BF16)
    if junk and ranks is not None:                                # what lies behind an adapter's rank is not used
        for i, r in enumerate(ranks):
            a[i, max(r, 0):] = float("nan")
            b[i, :, max(r, 0):] = float("nan")
    bs = torch.randn(M, N, generator=g, device="cuda").to(BF16) if base else None
    want_base = None if bs is None else bs.clone()
    sc = 2 * torch.randn(bank, generator=g, device="cuda") if scaling else None
    ad = torch.tensor(adapter, dtype=torch.int32, device="cuda")
    rk = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda")
    out = bs if in_place else torch.full((M, N), 9.0, dtype=BF16, device="cuda")
    serve.lora(L, x, a, b, ad, out, base=bs, scaling=sc, ranks=rk)
    torch.cuda.synchronize()
    assert L.device_error(True) == 0
    want, tol = C.lora(x, a, b, ad, want_base, sc, ranks)
    within(out, want, tol, (M, K, N, rank))
    return out


@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 40, 300])
@pytest.mark.parametrize("rank", [8, 16, 24, 64, 72, 256])
def test_lora_rows_and_ranks(L, M, rank):
    lora_case(L, M, 512, 640, rank, 5, [(3 * m) % 5 for m in range(M)])
    lora_case(L, M, 256, 264, rank, 3, [1] * M, seed=2)


@pytest.mark.parametrize("K,N", [(8, 8), (24, 40), (520, 1032), (4096, 6144), (14336, 264), (264, 28672)])
def test_lora_sizes(L, K, N):
    lora_case(L, 13, K, N, 16, 6, [m % 7 - 1 for m in range(13)])


def test_lora_rows_without_adapter_and_mixed_ranks(L):
    ranks = [0, 1, 7, 8, 9, 15, 16, 31, 32, -3, 100]
    adapter = [m % 12 - 1 for m in range(70)]
    lora_case(L, 70, 264, 520, 32, 11, adapter, ranks=ranks, junk=True)
    lora_case(L, 70, 264, 520, 32, 11, adapter, ranks=ranks, junk=True, base=False)
    lora_case(L, 70, 264, 520, 32, 11, adapter, ranks=ranks, junk=True, in_place=True)
    lora_case(L, 70, 264, 520, 32, 11, [-1] * 70)
    lora_case(L, 5, 264, 520, 32, 11, [-1] * 5, base=False)


def test_lora_many_adapters_and_rows(L):
    lora_case(L, 400, 128, 136, 8, 8192, [(m * 37) % 8192 for m in range(400)])
    lora_case(L, 3000, 64, 72, 8, 2, [(m * m) % 3 - 1 for m in range(3000)])


@pytest.mark.parametrize("M,bank,rank,ids", [
    (257, 1, 8, lambda m: 0), (2500, 3, 16, lambda m: m % 4 - 1), (6000, 1, 24, lambda m: 0),
    (5200, 700, 8, lambda m: m * m % 701 - 1), (9000, 300, 8, lambda m: 299 if m > 1000 else m % 7),
    (20000, 5, 72, lambda m: -1 if m % 11 else m % 5), (400, 8192, 256, lambda m: (m * 41) % 8192)])
def test_lora_prompt_rows(L, M, bank, rank, ids):
    """More items than CTAs: each takes a run of them, over adapters of one row and of thousands."""
    lora_case(L, M, 40, 24, rank, bank, [ids(m) for m in range(M)])


def test_lora_strided(L):
    from paia_gemv import serve
    g = gen(8)
    wide = torch.randn(10, 300 + 4, generator=g, device="cuda").to(BF16)
    x = torch.randn(10, 512, generator=g, device="cuda").to(BF16)[:, 128:384]
    a = (torch.randn(4, 20, 512, generator=g, device="cuda") / 16).to(BF16)[:, 2:18, 64:320]
    b = (torch.randn(4, 300, 24, generator=g, device="cuda") * 0.1).to(BF16)[:, 4:268, 8:24]
    y = torch.full((10, 400), 9.0, dtype=BF16, device="cuda")
    out = y[:, 64:328]
    base = wide[:, 8:272]
    ad = torch.tensor([0, 3, 3, -1, 2, 0, 0, 1, 2, 3], dtype=torch.int32, device="cuda")
    serve.lora(L, x, a, b, ad, out, base=base)
    want, tol = C.lora(x, a, b, ad, base)
    within(out, want, tol)
    assert (y[:, :64] == 9).all() and (y[:, 328:] == 9).all()


def test_lora_bad_ids_are_reported(L):
    """An id outside the bank is no adapter (code 13)."""
    from paia_gemv import serve
    g = gen(8)
    x = torch.randn(3, 64, generator=g, device="cuda").to(BF16)
    a, b = torch.ones(2, 8, 64, dtype=BF16, device="cuda"), torch.ones(2, 64, 8, dtype=BF16, device="cuda")
    base, out = torch.randn(3, 64, generator=g, device="cuda").to(BF16), torch.empty(3, 64, dtype=BF16, device="cuda")
    for bad in (2, -2, 0x7FFFFFFF):
        ad = torch.tensor([0, bad, 1], dtype=torch.int32, device="cuda")
        serve.lora(L, x, a, b, ad, out, base=base)
        assert L.device_error(True) == 13 and torch.equal(out[1], base[1])
        want, tol = C.lora(x, a, b, ad, base)
        within(out, want, tol)


def test_lora_same_bits_whoever_shares_the_batch(L):
    """A row's result does not depend on the rows beside it of the same call, nor on the run."""
    one = lora_case(L, 12, 520, 520, 16, 4, [2] * 12)
    for _ in range(3):
        assert torch.equal(one, lora_case(L, 12, 520, 520, 16, 4, [2] * 12))


@pytest.mark.parametrize("M", [33, 37, 43, 52, 65, 86, 129, 148, 149])
@pytest.mark.parametrize("rank", [16, 256])
def test_lora_every_cluster_size(L, M, rank):
    """As many adapters as rows: 8 CTAs per item down to one, with K and N that do not divide by them."""
    lora_case(L, M, 1000, 1208, rank, M, [(7 * m) % M for m in range(M)])
