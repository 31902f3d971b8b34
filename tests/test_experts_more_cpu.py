"""CPU (no GPU needed): what the kernels of a block with experts promise one another inside, from the source, and refusals at
the ends of the sizes."""
import re

from test_experts_cpu import code


def test_gathering_warps_read_their_list_behind_a_barrier():
    """expert_kernel: the lanes of a gathering warp write where their rows begin and read what other lanes wrote; votes order no
    memory, so a warp barrier stands between the last write and the first read, and between the reads and the next list."""
    src = code("block_experts.cu")
    body = src[src.index("const __nv_bfloat16** list ="):src.index("cp_arrive(")]
    write, read = body.index("list[r] ="), re.search(r"list\[r\](?! =)", body).start()
    assert body.count("list[r] =") == 1 and write < read
    assert "__syncwarp();" in body[body.index("walk.next(s)"):write]
    assert "__syncwarp();" in body[write:read]
