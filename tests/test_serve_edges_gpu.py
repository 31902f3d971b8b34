"""The serving operators at the edges of what they take: errors beside one another, batches beyond the size that one scan
finds its place in, infinities and NaN."""

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
