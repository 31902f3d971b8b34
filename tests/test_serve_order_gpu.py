"""Runs of GEMVs and serving operators on one stream, each launched while the one before it finishes: what a kernel further
back has written is there for the weights and the bias that a GEMV reads ahead of its wait."""
import pytest
import torch

from serve_cases import BF16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from paia_gemv import load_lib
    lib = load_lib()
    lib.device_error(True)
    return lib


def operators(L, g):
    """The three operators at sizes that take a few microseconds, each on tensors of its own."""
    from paia_gemv import serve
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF16)   # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    q, out, pool, ws = r(2, 8, 64), r(2, 8, 64), r(9, 16, 2, 64), serve.attention_workspace(L, 8, 2, 64)
    table, lens = i32([[0, 1, 2], [3, 4, 5]]), i32([40, 7])
    positions = i32([3, 17])
    qkv, freq, q2, k, v = r(2, 12 * 64), serve.rope_inv_freq(64, 1e4), r(2, 8, 64), r(9, 16, 2, 64), r(9, 16, 2, 64)
    x, a, b, y, ad = r(3, 64), r(2, 8, 64), r(2, 64, 8), r(3, 64), i32([0, 1, -1])
    return {"attention": lambda: serve.paged_attention(L, q, pool, pool, table, lens, out, ws),
            "rope": lambda: serve.qkv_rope_cache(L, qkv, positions, freq, q2, k, v, table),
            "lora": lambda: serve.lora(L, x, a, b, ad, y)}


@pytest.mark.parametrize("between", ["attention", "rope", "lora", "all"])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_bias_written_two_kernels_back(L, between, kind):
    """A long GEMV writes y; an operator that has nothing to do with it follows; a GEMV adds y as its bias."""
    g = torch.Generator(device="cuda").manual_seed(5)
    ops = operators(L, g)
    run = [ops[between]] if between != "all" else list(ops.values())
    n, k, small = 28672, 4096, 1024
    W = (torch.randn(n, k, generator=g, device="cuda") * 0.02).to(BF16)
    V = (torch.randn(n, small, generator=g, device="cuda") * 0.02)
    V8, s = V.to(torch.float8_e4m3fn), torch.ones(n, device="cuda")
    V = V.to(BF16)
    xs = [torch.randn(k, generator=g, device="cuda").to(BF16) for _ in range(2)]
    x2 = torch.randn(small, generator=g, device="cuda").to(BF16)
    y, z = torch.zeros(n, dtype=BF16, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    pick = lambda table: next(e["id"] for e in table if e["H"] == 1 and e["R"] == 2)   # noqa: E731
    v16, v8 = pick(L.variants), pick(L.variants_fp8)

    def first(i):
        L.bf16(W.data_ptr(), xs[i].data_ptr(), y.data_ptr(), n, k, v16)

    def last():
        if kind == "bf16":
            L.bf16_bias(V.data_ptr(), x2.data_ptr(), y.data_ptr(), z.data_ptr(), n, small, v16)
        else:
            L.fp8_bias(V8.data_ptr(), s.data_ptr(), x2.data_ptr(), y.data_ptr(), z.data_ptr(), n, small, v8)

    want = []
    for i in range(2):
        first(i)
        torch.cuda.synchronize()
        last()
        torch.cuda.synchronize()
        want.append(z.clone())
    assert not torch.equal(want[0], want[1])
    for t in range(30):
        first(t % 2)
        for op in run:
            op()
        last()
        got = z.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want[t % 2]), t
    assert L.device_error(True) == 0
