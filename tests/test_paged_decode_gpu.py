"""The batched decode step over a paged cache (paia_gemv.decode.PagedDecodeModel): batched GEMVs, adapters, rotary and
cache write, paged attention run together, against the same arithmetic in plain torch fp32 on the same bytes, token after
token with growing lengths; captured in a graph; with padding rows."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DIMS = dict(hidden=512, heads=8, kv_heads=2, head_dim=64, inter=1024, vocab=1000, layers=2, qkv_bias=True)


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paia_gemv import load_lib
    return load_lib()


class Plain:
    """The step in fp32 torch with the roundings of the bf16 activations between its parts; its own dense cache."""

    def __init__(self, m):
        self.m, c = m, m.cfg
        nkv, hd = c["kv_heads"], c["head_dim"]
        self.cache = []
        for lay in m.layers:
            kv = []
            for name, sc in (("k", m.k_scale), ("v", m.v_scale)):
                x = lay[name][m.page_table.long()].float().flatten(1, 2)          # [batch, positions, kv, hd]
                kv.append(x if sc is None else x * sc.view(1, 1, nkv, 1))
            self.cache.append(kv)
        self.lens = m.lens.tolist()

    @staticmethod
    def norm(x, w, eps):
        return F.rms_norm(x.float(), (x.shape[-1],), w, eps)

    def project(self, lay, name, x):
        m = self.m
        y = x.float() @ lay[name].dequantised().float().T
        if lay[name].bias is not None:
            y = y + lay[name].bias.float()
        y = y.bfloat16()
        if m.adapter is not None:
            y = y.float()
            for b, i in enumerate(m.adapter.tolist()):
                if i >= 0:
                    y[b] += (x[b].float() @ lay[name + "_a"][i].float().T) @ lay[name + "_b"][i].float().T
            y = y.bfloat16()
        return y

    def turn(self, x, pos):
        half = x.shape[-1] // 2
        ang = pos * self.m.inv_freq
        c, s = ang.cos().float(), ang.sin().float()
        return torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)

    def step(self, token):
        m, c = self.m, self.m.cfg
        nh, nkv, hd, I = c["heads"], c["kv_heads"], c["head_dim"], c["inter"]
        h = m.embed[token]
        for lay, (ck, cv) in zip(m.layers, self.cache):
            qkv = self.project(lay, "qkv", self.norm(h, lay["norm1"], 1e-5).bfloat16()).float().view(-1, nh + 2 * nkv, hd)
            att = torch.zeros(len(self.lens), nh, hd, device=h.device)
            for b, n in enumerate(self.lens):
                if n is None:
                    continue
                q, k, v = qkv[b, :nh], qkv[b, nh:nh + nkv], qkv[b, nh + nkv:]
                if lay["q_norm"] is not None:
                    q, k = self.norm(q, lay["q_norm"], 1e-6), self.norm(k, lay["k_norm"], 1e-6)
                q, k = self.turn(q, n).bfloat16().float(), self.turn(k, n)
                if m.k_scale is None:
                    ck[b, n], cv[b, n] = k.bfloat16().float(), v
                else:
                    q8 = lambda x, s: (x / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s[:, None]   # noqa: E731
                    ck[b, n], cv[b, n] = q8(k, m.k_scale), q8(v, m.v_scale)
                kk = ck[b, :n + 1].repeat_interleave(nh // nkv, 1)
                vv = cv[b, :n + 1].repeat_interleave(nh // nkv, 1)
                p = torch.softmax(torch.einsum("hd,lhd->hl", q, kk) * hd ** -0.5, -1)
                att[b] = torch.einsum("hl,lhd->hd", p, vv)
            h = h + self.project(lay, "o", att.bfloat16().flatten(1))
            gu = self.project(lay, "gate_up", self.norm(h, lay["norm2"], 1e-5).bfloat16())
            h = h + self.project(lay, "down", F.silu(gu[:, :I]) * gu[:, I:])
        self.lens = [n if n is None else n + 1 for n in self.lens]
        return self.norm(h, m.norm_f, 1e-5).bfloat16().float() @ m.lm_head.dequantised().float().T


def rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("kind,cache,adapters,qk_norm", [("bf16", "bf16", 0, False), ("fp8", "bf16", 3, True),
                                                        ("int4", "fp8", 3, False), ("int4_asym", "fp8", 0, True)])
def test_paged_step_matches_plain_torch(L, kind, cache, adapters, qk_norm):
    from paia_gemv import decode
    m = decode.PagedDecodeModel(L, "qwen25_7b", kind, lens=[0, 15, 31, 100, 7], max_len=128, cache=cache,
                                adapters=adapters, qk_norm=qk_norm, dims=DIMS, seed=3)
    if adapters:
        m.adapter.copy_(torch.tensor([0, 2, -1, 2, 1], dtype=torch.int32))
    ref = Plain(m)
    # 1e-2 as for the unbatched step (bf16 activations between the parts). An e4m3 cache adds what a bf16 difference of the
    # projections does to the rows that are stored: GEMV and plain product agree to 1e-3 (relative L2, the bar of the GEMV
    # tests), that is (1e-3 / (0.72 * 2^-8))^2 = 0.126 of the values one bf16 step apart (a step is 0.72 * 2^-8 of the
    # value on average, rms over the mantissas); one in 16 of those steps crosses a border between e4m3 values (16 bf16
    # steps each), which moves the value by 0.72 * 2^-3: 0.09 * sqrt(0.126 / 16) = 8e-3 of v in each of the two layers.
    tol = 1e-2 if cache == "bf16" else (1e-2 ** 2 + 2 * 8e-3 ** 2) ** 0.5
    for t in range(4):
        tok = torch.tensor([17 + t, 3, 500, 999 - t, 3], device="cuda")
        m.token.copy_(tok)
        a = m.step().clone()
        b = ref.step(tok)
        torch.cuda.synchronize()
        for i in range(5):
            assert rel(a[i], b[i]) < tol, (kind, t, i)
        assert m.lens.tolist() == ref.lens
    assert L.device_error(True) == 0


def test_paged_step_graph_and_padding(L):
    """Replays of one captured step decode token after token as eager steps do; rows set inactive keep cache and length."""
    from paia_gemv import decode

    def make():
        return decode.PagedDecodeModel(L, "llama31_8b", "fp8", lens=[5, 40, 16], max_len=64, adapters=2,
                                       dims=dict(DIMS, qkv_bias=False), seed=5)

    a, b = make(), make()
    for m in (a, b):
        m.adapter.copy_(torch.tensor([1, -1, 0], dtype=torch.int32))
    b.step()                                                     # warm-up, then back to the start
    b.token.zero_()
    b.lens.copy_(a.lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.step()
    for t in range(6):
        if t == 3:
            for m in (a, b):
                m.active[1] = False
        a.step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.token, b.token) and torch.equal(a.lens, b.lens)
        assert torch.equal(a.logits[[0, 2]], b.logits[[0, 2]])
    assert a.lens.tolist() == [11, 43, 22]
    for la, lb in zip(a.layers, b.layers):
        assert torch.equal(la["k"], lb["k"]) and torch.equal(la["v"], lb["v"])
    assert L.device_error(True) == 0


def test_paged_model_refuses_bad_lengths(L):
    from paia_gemv import decode
    for lens in ([], [64], [-1, 3]):
        with pytest.raises(ValueError):
            decode.PagedDecodeModel(L, "llama31_8b", "bf16", lens=lens, max_len=64, dims=DIMS)
