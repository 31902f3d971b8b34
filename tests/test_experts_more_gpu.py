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
