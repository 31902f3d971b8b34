"""What a serving operator promises the kernels around it on the stream, under programmatic dependent launch: it triggers
the next kernel only behind its own wait, and reads by loads that see what the kernel before it wrote. (On the CPU: from the
source.)"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "paia-project_b200" / "csrc"


def code(name):
    """A source without its comments."""
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_trigger_comes_after_the_wait():
    """A kernel that triggered before it has waited would let the next one start while kernels further back still run; a
    GEMV reads its weights and bias before its own wait and is promised that all but the kernel before it are done."""
    common = code("serve_common.cuh")
    at = [m.start() for m in re.finditer(r"griddepcontrol\.(wait|launch_dependents)", common)]
    assert len(at) == 2 and common.index("griddepcontrol.wait") < common.index("griddepcontrol.launch_dependents")
    for name in ("serve_attn.cu", "serve_rope.cu", "serve_lora.cu"):
        src = code(name)
        assert "griddepcontrol" not in src, name
        kernels = [m.end() for m in re.finditer(r"__global__", src)]
        assert kernels and len(re.findall(r"\bpdl_wait_and_trigger\(\);", src)) == len(kernels), name
        for at in kernels:                                       # before any way out of the kernel
            body = src[at:]
            head = body[:body.index("pdl_wait_and_trigger();")]
            assert not re.search(r"\breturn;", re.sub(r"\[&\]\([^)]*\) \{.*?\n    \};", "", head, flags=re.S)), name


def test_no_load_promises_unchanged_memory():
    """The kernels live while the kernel before them still writes lengths, page tables, queries, positions and adapter ids:
    the read-only path is not for them, neither asked for nor left to the compiler (restrict)."""
    for name in ("serve_common.cuh", "serve_attn.cu", "serve_rope.cu", "serve_lora.cu"):
        assert not re.search(r"__ldg|\.nc\b|__restrict", code(name)), name


def test_gemv_reads_x_plainly():
    """The same holds for x of the GEMVs, which is read behind their wait. (Weights, scales and bias are read ahead of it and
    are the caller's to leave alone: their loads take the read-only path, in helpers that know nothing of x.)"""
    for name in ("gemv_kernel.cuh", "gemv_mma.cuh", "gemv_tma.cuh"):
        assert "__ldg" not in code(name), name
