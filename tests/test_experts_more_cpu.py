"""CPU (no GPU needed): what the kernels of a block with experts promise one another inside, from the source, and refusals at
the ends of the sizes."""
import re

import torch

from test_experts_cpu import L, code  # noqa: F401  (a fixture among them)


def test_gathering_warps_read_their_list_behind_a_barrier():
    """expert_kernel: the lanes of a gathering warp write where their rows begin and read what other lanes wrote; votes order no
    memory, so a warp barrier stands between the last write and the first read, and between the reads and the next list."""
    src = code("block_experts.cu")
    body = src[src.index("const __nv_bfloat16** list ="):src.index("cp_arrive(")]
    write, read = body.index("list[r] ="), re.search(r"list\[r\](?! =)", body).start()
    assert body.count("list[r] =") == 1 and write < read
    assert "__syncwarp();" in body[body.index("walk.next(s)"):write]
    assert "__syncwarp();" in body[write:read]


def test_four_e4m3_terms_of_every_bf16():
    """split_kernel: v below 2^8 as t0 + t1 + 2^-16 (t2 + t3), each e4m3 and the nearest to what is left. From 2^-18 on nothing is
    left, below at most 2^-26, and up to 2^-26 there are no terms."""
    v = torch.arange(0x0080, 0x4380, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).double()
    assert v.max() < 256 and v.min() == 2.0 ** -126
    left, terms = v.clone(), []
    for t in range(4):
        if t == 2:
            left = left * 2.0 ** 16
        assert left.abs().max() <= 448                           # nothing saturates
        terms.append(left.float().to(torch.float8_e4m3fn).double())
        left = left - terms[-1]
    left = left * 2.0 ** -16
    assert torch.equal(terms[0] + terms[1] + (terms[2] + terms[3]) * 2.0 ** -16 + left, v)
    assert not left[v >= 2.0 ** -18].any() and left.abs().max() <= 2.0 ** -26
    none = sum(t.abs() for t in terms) == 0
    assert torch.equal(none, v <= 2.0 ** -26)


def test_terms_and_marks_fit_the_workspace(L):
    """The largest calls whose x enters as terms: 4 K bytes and a word per row, then a word for every 256 of K."""
    src = code("block_experts.cu")
    number = lambda name: int(re.search(rf"constexpr (?:int|size_t) {name} = (\d+)", src).group(1))   # noqa: E731
    tokens, experts, split = number("kExpSplitTokens"), number("kExpMaxExperts"), number("kExpSplitBytes") << 20
    assert re.search(r"kExpSplitBytes = 48 << 20;", src) and re.search(r"want <= 2 \* kExpSplitTokens", src)
    room = L.expert_workspace() - 2 * 160 * 4 - 2 * 160 * 128 * 256 * 4      # counters, parts
    for k in [16 * i for i in range(1, 400)] + [256 * i + d for i in (30, 500, 4095) for d in (-16, 0, 16)] + [1 << 20]:
        m = min(split // (4 * k + 4), tokens * experts)
        assert m * (4 * k + 4) + m * 4 * -(-k // 256) <= room, (k, m)


def test_sizes_whose_tiles_pass_an_int_are_refused(L):
    """Rows of W are counted in tiles of up to 256, and a tile's last rows may lie behind N: both within an int."""
    from paia_gemv import serve
    from test_experts_cpu import EXPERTS, packed
    most = re.search(r"a->N > (\d+) << (\d+)", code("block_experts.cu"))
    assert most and (int(most.group(1)) << int(most.group(2))) + 2 * 255 < 2 ** 31
    big = dict(N=2 ** 31 - 200, K=8, w_row=8, w_expert=8 * (2 ** 31 - 200), out_row=2 ** 31 - 200)
    assert L._lib.paia_gemv_expert_matmul(packed("paia_gemv_expert_args", serve.EXPERTS, EXPERTS, **big), None) == -2


def test_norm_counts_rows_without_passing_an_int():
    """block_norm_kernel steps by the grid's size from its last row, of up to 2^31 - 1: in an unsigned."""
    src = code("block_norm.cu")
    loop = re.search(r"for \((\w+) t = blockIdx\.x; t < (\w+(?:\.\w+)?); t \+= gridDim\.x\)", src)
    assert loop and loop.group(1) == "unsigned" and re.search(rf"const unsigned {loop.group(2)} = p\.tokens;", src)
    assert "(int)gridDim.x" not in src[src.index("block_norm_kernel"):src.index("launch_norm")]
