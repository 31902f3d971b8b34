"""The batched decode step with experts (paia_gemv.decode.PagedDecodeModel, experts > 0): routing, grouped products and block norms
run together with the batched GEMVs, the rotary and cache write and the paged attention, against the same arithmetic in plain
torch fp32 on the same bytes; captured in a graph, with padding rows."""
import pytest
import torch
import torch.nn.functional as F

from paia_gemv import quant
from test_paged_decode_gpu import DIMS, Plain, rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paia_gemv import load_lib
    return load_lib()


class PlainExperts(Plain):
    """The plain step whose feed-forward block is experts: `ids`, where given, is each row's choice."""

    ids = None

    def expert(self, lay, name, e):
        w, s = lay[name][e], lay[name + "_s"]
        return w.float() if s is None else quant.dequant_fp8(w, s[e])

    def project(self, lay, name, x):
        m = self.m
        if name == "down":
            return self.block
        if name != "gate_up":
            y = super().project(lay, name, x)
            return self.norm(y, lay["post1"], 1e-5).bfloat16() if name == "o" and lay["post1"] is not None else y
        logits = (x.float() @ lay["router"].float().T).bfloat16().float()
        k = m.routing.sizes[3]
        ids = torch.topk(logits, k, 1).indices if self.ids is None else self.ids
        chosen = logits.gather(1, ids)
        # a choice that is given: within a few bf16 steps of the largest
        assert bool((chosen.amin(1) >= logits.topk(k, 1).values[:, -1] - 0.1).all())
        w = torch.softmax(chosen, 1) if m.scoring == "softmax" else torch.sigmoid(chosen) / torch.sigmoid(chosen).sum(1, True)
        y = torch.zeros(x.shape[0], m.cfg["hidden"], device=x.device)
        for b in range(x.shape[0]):
            for j in range(k):
                g, u = (self.expert(lay, "experts_gate_up", ids[b, j]) @ x[b].float()).chunk(2)
                y[b] += w[b, j] * (self.expert(lay, "experts_down", ids[b, j]) @ (F.silu(g) * u).bfloat16().float()).bfloat16()
        self.block = y if lay["post2"] is None else self.norm(y, lay["post2"], 1e-5)
        self.block = self.block.bfloat16()
        return torch.zeros(x.shape[0], 2 * m.cfg["inter"], device=x.device, dtype=torch.bfloat16)


@pytest.mark.parametrize("kind,experts,top_k,layers,scoring,post", [
    ("bf16", 4, 4, 2, "softmax", False), ("fp8", 4, 4, 2, "sigmoid", True), ("fp8", 8, 2, 1, "softmax", False),
    ("bf16", 16, 3, 1, "sigmoid", True)])
def test_step_matches_plain_torch(L, kind, experts, top_k, layers, scoring, post):
    from paia_gemv import decode
    m = decode.PagedDecodeModel(L, "qwen25_7b", kind, lens=[0, 15, 31, 100, 7], max_len=128, adapters=2, qk_norm=True,
                                dims=dict(DIMS, layers=layers), seed=3, experts=experts, top_k=top_k, expert_inter=192,
                                scoring=scoring, post_norm=post)
    m.adapter.copy_(torch.tensor([0, 1, -1, 1, -1], dtype=torch.int32))
    ref = PlainExperts(m)
    for t in range(3):
        tok = torch.tensor([17 + t, 3, 500, 999 - t, 3], device="cuda")
        m.token.copy_(tok)
        a = m.step().clone()
        if layers == 1:
            ref.ids = m.routing.experts.long().clone()
        b = ref.step(tok)
        torch.cuda.synchronize()
        for i in range(5):
            assert rel(a[i], b[i]) < 1e-2, (t, i)                # as for the step without experts
        assert m.lens.tolist() == ref.lens
    assert L.device_error(True) == 0


def test_graph_and_padding(L):
    """Replays of one captured step decode as eager steps do; an inactive row takes no expert's time and keeps its cache."""
    from paia_gemv import decode

    def make():
        return decode.PagedDecodeModel(L, "llama31_8b", "fp8", lens=[5, 40, 16], max_len=64, dims=dict(DIMS, qkv_bias=False),
                                       seed=5, experts=8, top_k=2, expert_inter=256)

    a, b = make(), make()
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
        assert torch.equal(a.logits, b.logits)
        assert int(a.routing.offsets[-1]) == (6 if t < 3 else 4)
    assert a.lens.tolist() == [11, 43, 22]
    assert L.device_error(True) == 0


def test_refuses_int4_experts(L):
    from paia_gemv import decode
    with pytest.raises(ValueError):
        decode.PagedDecodeModel(L, "llama31_8b", "int4", lens=[3], max_len=64, dims=DIMS, experts=4)
