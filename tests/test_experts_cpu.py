"""CPU (no GPU needed): the C structs of the operators of a block with experts as paia_gemv.serve packs them, their refusals on
the host (code -2 before any device is touched), the checks of the tensor wrappers, what their kernels promise on a stream (from
the source), and a replay of how expert_matmul's tiles are divided."""
import random
import re
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "paia-project_b200" / "csrc"
PTR = 0x10000


@pytest.fixture(scope="module")
def L(lib_path):
    from paia_gemv import loader
    return loader.GemvLib(lib_path)


def fields(name):
    txt = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "paia_gemv.h").read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, txt, flags=re.S).group(1)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind = "P" if "*" in decl else "q" if decl.startswith("long long") else "f" if decl.startswith("float") else "i"
        names = re.sub(r"^(const )?(void|int|float|long long)\b", "", decl)
        out += [(n.strip(" *"), kind) for n in names.split(",")]
    return out


def packed(name, fmt, good, **change):
    values = dict(good, **change)
    assert {n for n, _ in fields(name)} == set(values)
    return fmt.pack(*[values[n] for n, _ in fields(name)])


ROUTE = dict(logits=PTR, bias=0, pos=0, weights=PTR, ids=PTR, places=PTR, rows=PTR, offsets=PTR, workspace=PTR, logits_row=8,
             tokens=3, experts=8, top_k=2, logits_type=0, scoring=0, renormalise=1, scale=1.0)
EXPERTS = dict(w=PTR, scales=0, x=PTR, rows=0, offsets=PTR, out=2 * PTR, workspace=PTR, w_expert=4096, w_row=64, x_row=64,
               out_row=64, scale_expert=0, experts=2, M=3, N=64, K=64, x_rows=3, kind=0, silu=0, pad=0)
NORM = dict(x=PTR, h=2 * PTR, h_out=3 * PTR, out=4 * PTR, places=0, weights=0, post=0, pre=PTR, gate=0, x_row=64, h_row=64,
            h_out_row=64, out_row=64, places_row=0, weights_row=0, gate_row=0, tokens=3, hidden=64, top_k=0, x_rows=3, gate_col=0,
            eps=1e-5, scale=1.0, pad=0)


def test_structs_match_the_header(tmp_path):
    from paia_gemv import serve
    names = {"paia_gemv_route_args": serve.ROUTE, "paia_gemv_expert_args": serve.EXPERTS,
             "paia_gemv_block_norm_args": serve.BLOCK_NORM}
    for n, fmt in names.items():
        kinds = "".join(k for _, k in fields(n))
        assert kinds == "".join(k * int(c or 1) for c, k in re.findall(r"(\d*)([Pqif])", fmt.format)), n
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "paia_gemv.h"\nint main(void) { printf("%zu %zu %zu", '
                   + ", ".join(f"sizeof({n})" for n in names) + "); return 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [f.size for f in names.values()]


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=9),
    dict(experts=64, top_k=33), dict(logits_type=2), dict(scoring=2), dict(scoring=-1), dict(bias=PTR), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(logits=0), dict(weights=0), dict(ids=0), dict(places=0), dict(rows=0), dict(offsets=0),
    dict(workspace=0), dict(logits=PTR + 1), dict(logits_type=1, logits=PTR + 2), dict(scoring=1, bias=PTR + 2),
    dict(pos=PTR + 1), dict(weights=PTR + 2), dict(ids=PTR + 2), dict(places=PTR + 1), dict(rows=PTR + 3), dict(offsets=PTR + 2),
    dict(workspace=PTR + 8)])
def test_route_refusals(L, change):
    from paia_gemv import serve
    assert L._lib.paia_gemv_route(packed("paia_gemv_route_args", serve.ROUTE, ROUTE, **change), None) == -2


@pytest.mark.parametrize("change", [
    dict(experts=0), dict(experts=1025), dict(M=-1), dict(M=(1 << 28) + 1), dict(N=0), dict(K=0), dict(K=60), dict(K=1 << 21),
    dict(kind=2), dict(kind=-1), dict(kind=1), dict(scales=PTR), dict(kind=1, scales=PTR, K=72), dict(silu=1, N=63), dict(w=0),
    dict(x=0), dict(offsets=0), dict(out=0), dict(workspace=0), dict(w=PTR + 8), dict(x=PTR + 8), dict(out=2 * PTR + 1),
    dict(rows=PTR + 2), dict(offsets=PTR + 1), dict(kind=1, scales=PTR + 2), dict(workspace=PTR + 8), dict(w_row=68),
    dict(w_row=56), dict(w_expert=4100), dict(w_expert=0), dict(x_row=60), dict(x_rows=2), dict(x_rows=-1), dict(out_row=0),
    dict(out=PTR), dict(rows=PTR, x_rows=0), dict(kind=1, scales=PTR, w_row=72)])
def test_expert_refusals(L, change):
    from paia_gemv import serve
    assert L._lib.paia_gemv_expert_matmul(packed("paia_gemv_expert_args", serve.EXPERTS, EXPERTS, **change), None) == -2


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(hidden=0), dict(hidden=60), dict(hidden=32776), dict(top_k=-1), dict(top_k=65), dict(eps=-1.0),
    dict(eps=float("nan")), dict(scale=float("inf")), dict(h=0), dict(h_out=0, out=0, pre=0), dict(out=0), dict(pre=0),
    dict(h_out=0), dict(x=0), dict(x=0, h_out=0, gate=PTR), dict(x=0, h_out=0, post=PTR), dict(x=0, h_out=0, out=0, pre=0),
    dict(top_k=2), dict(top_k=2, places=PTR), dict(places=PTR), dict(weights=PTR), dict(x_rows=2), dict(x=PTR + 8),
    dict(h=2 * PTR + 2), dict(h_out=3 * PTR + 4), dict(out=4 * PTR + 8), dict(post=PTR + 4), dict(pre=PTR + 8),
    dict(top_k=2, places=PTR + 2, weights=PTR), dict(top_k=2, places=PTR, weights=PTR + 1), dict(gate=PTR + 1),
    dict(gate=PTR + 2, gate_col=1), dict(gate=PTR, gate_col=2), dict(gate=PTR, gate_col=1, gate_row=4), dict(x_row=60),
    dict(h_row=4), dict(h_out_row=0), dict(out_row=0), dict(out_row=12), dict(out=2 * PTR), dict(out=3 * PTR), dict(out=PTR),
    dict(h_out=PTR)])
def test_block_norm_refusals(L, change):
    from paia_gemv import serve
    assert L._lib.paia_gemv_block_norm(packed("paia_gemv_block_norm_args", serve.BLOCK_NORM, NORM, **change), None) == -2


def test_nothing_to_do(L):
    from paia_gemv import serve
    assert L._lib.paia_gemv_expert_matmul(packed("paia_gemv_expert_args", serve.EXPERTS, EXPERTS, M=0, x=0, out=0), None) == 0
    assert L._lib.paia_gemv_block_norm(packed("paia_gemv_block_norm_args", serve.BLOCK_NORM, NORM, tokens=0), None) == 0
    assert L._lib.paia_gemv_route(None, None) == -2 and L._lib.paia_gemv_block_norm(None, None) == -2
    assert L._lib.paia_gemv_expert_matmul(None, None) == -2
    assert L._lib.paia_gemv_route_workspace(0) == 0 == L._lib.paia_gemv_route_workspace(1025)
    with pytest.raises(RuntimeError):
        L.route_workspace(2000)
    assert L.expert_workspace() > 0


def test_wrappers_refuse_cpu_tensors(L):
    from paia_gemv import serve
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)   # noqa: E731
    r = serve.Routing(L, torch.zeros(4, 2), *(torch.zeros(*s, dtype=torch.int32) for s in ((4, 2), (4, 2), (8,), (9,))),
                      torch.zeros(0, dtype=torch.uint8))
    assert r.first(3).sizes == (-1, 3, 8, 2)
    with pytest.raises(ValueError):
        serve.route(L, bf(4, 8), r)
    with pytest.raises(ValueError):
        serve.Routing(L, torch.zeros(4, 2), *(torch.zeros(*s, dtype=torch.int32) for s in ((4, 3), (4, 2), (8,), (9,))),
                      torch.zeros(0, dtype=torch.uint8))
    ws = serve.ExpertWorkspace(torch.zeros(16, dtype=torch.uint8))
    with pytest.raises(ValueError):
        serve.expert_matmul(L, bf(2, 8, 8), bf(4, 8), torch.zeros(3, dtype=torch.int32), bf(4, 8), ws)
    with pytest.raises(ValueError):
        serve.block_norm(L, bf(4, 8), out=bf(4, 8), pre=torch.zeros(8))


def code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_stream_order():
    """As every serving operator: each kernel waits for the one before it before anything that a caller may have written is
    read, lets the next one start only then, and asks for no load through the read-only path."""
    for name in ("block_route.cu", "block_experts.cu", "block_norm.cu"):
        src = code(name)
        kernels = [m.end() for m in re.finditer(r"__global__", src)]
        # (expert_kernel behind its own split_kernel waits where it reads what that writes)
        late = len(re.findall(r"if \(FMT == kSplit\) pdl_wait_and_trigger\(\);", src))
        assert kernels and len(re.findall(r"\bpdl_wait_and_trigger\(\);", src)) == len(kernels) + late, name
        assert late == (2 if name == "block_experts.cu" else 0)
        assert "griddepcontrol" not in src and not re.search(r"__ldg|\.nc\b|__restrict", src), name
        for at in kernels:
            head = src[at:][:src[at:].index("pdl_wait_and_trigger();")]
            assert not re.search(r"\breturn;", head), name


# ------------------------------------------------------------------ the division of tiles

def walk(counts, tokens, row_tiles, units, grid, cg, min_run):
    """What each CTA (pair) of expert_kernel works on: [(tile, k0, k1, expert, row tile, first row, rows)], as ExpWalk has it."""
    first, off = [0], [0]
    for c in counts:
        first.append(first[-1] + -(-c // tokens) * row_tiles)
        off.append(off[-1] + c)
    g = grid // cg
    total = first[-1]
    rounds = total // g
    cut = total - rounds * g
    if cut and rounds:
        cut += g
    elif 4 * cut >= 3 * g:
        cut = 0
    work = cut * units
    workers = min(g, max(cut, 1, work // min_run))
    if rounds == 0 and cut:
        workers -= workers % cut
    bound = lambda c: c * work // workers                        # noqa: E731
    parts = []
    for c in range(g):
        mine = []
        at, end = (bound(c), bound(c + 1)) if c < workers else (0, 0)
        while at < end:
            tile = at // units
            k0 = at - tile * units
            k1 = min(units, k0 + end - at)
            mine.append((tile, k0, k1))
            at += k1 - k0
        mine += [(t, 0, units) for t in range(cut + c, total, g)]
        out = []
        for tile, k0, k1 in mine:
            e = max(i for i in range(len(counts)) if first[i] <= tile)
            assert first[e] <= tile < first[e + 1]
            blocks = (first[e + 1] - first[e]) // row_tiles
            local, step = tile - first[e], 16 * cg
            per = -(-(-(-counts[e] // blocks)) // step) * step
            row_tile, b = divmod(local, blocks)
            out.append((tile, k0, k1, e, row_tile, off[e] + b * per, min(per, counts[e] - b * per)))
        parts.append(out)
    owner = lambda u: ((u + 1) * workers - 1) // work            # noqa: E731
    place = lambda c, tile: 2 * c + (tile != bound(c) // units)  # noqa: E731
    return parts, total, cut, owner, place


def test_tiles_are_divided_once():
    src = code("block_experts.cu")
    min_run = int(re.search(r"kExpMinRun = (\d+)", src).group(1))
    rng = random.Random(5)
    for _ in range(300):
        e, cg = rng.choice([1, 2, 7, 40]), rng.choice([1, 2])
        counts = [rng.choice([0, 1, 3, 16, 17, 100, 700]) for _ in range(e)]
        tokens = rng.choice([16, 64, 128] if cg == 1 else [192, 256])
        row_tiles, units, grid = rng.choice([1, 3, 16, 40]), rng.choice([1, 2, 9, 56, 224]), rng.choice([148, 16])
        parts, total, cut, owner, place = walk(counts, tokens, row_tiles, units, grid, cg, min_run)
        seen, slots, arrivals = {}, set(), {}
        for c, mine in enumerate(parts):
            for tile, k0, k1, ex, rt, row0, m in mine:
                assert 0 <= k0 < k1 <= units and 1 <= m <= tokens and 0 <= rt < row_tiles
                assert sum(counts[:ex]) <= row0 and row0 + m <= sum(counts[:ex + 1])
                seen.setdefault(tile, []).append((k0, k1, c))
                if (k0, k1) != (0, units):
                    assert tile < cut < 2 * (grid // cg) + 1     # a counter of its own
                    slot = place(c, tile)
                    assert slot not in slots and slot < 2 * (grid // cg)
                    slots.add(slot)
                    arrivals.setdefault(tile, []).append(c)
        assert sorted(seen) == list(range(total))
        rows = {}
        for tile, ks in seen.items():
            ks.sort()
            assert ks[0][0] == 0 and ks[-1][1] == units and all(a[1] == b[0] for a, b in zip(ks, ks[1:]))
            if tile in arrivals:                                 # the parts that the last arrival joins are all there are
                assert sorted(arrivals[tile]) == list(range(owner(tile * units), owner((tile + 1) * units - 1) + 1))
        for mine in parts:
            for tile, k0, _, ex, rt, row0, m in mine:
                if k0 == 0:
                    rows.setdefault((ex, rt), []).append((row0, m))
        for (ex, rt), blocks in rows.items():                    # every row of an expert meets every tile of its weights once
            blocks.sort()
            assert blocks[0][0] == sum(counts[:ex]) and all(a + n == b for (a, n), (b, _) in zip(blocks, blocks[1:]))
            assert sum(n for _, n in blocks) == counts[ex]
        assert len(rows) == sum(c > 0 for c in counts) * row_tiles


def test_registers():
    """ptxas's report: nothing of the products' kernels spills, and a CTA's registers fit the SM at its size."""
    from test_compile_report import load_reports
    rows = [r for r in load_reports() if r["file"].startswith("block_")]
    threads = {0: 384, 1: 384, 2: 896}                           # bf16, split, converted
    seen = 0
    for r in rows:
        m = re.search(r"expert_kernelILi(\d)ELb(\d)ELi(\d)E", r["fn"])
        if m:
            seen += 1
            assert r["regs"] * threads[int(m.group(1))] <= 65536 and r["spill_st"] + r["spill_ld"] <= 64, r
        if "block_norm_kernel" in r["fn"] or "route_place" in r["fn"]:
            assert r["spill_st"] == 0 and r["stack"] == 0, r
    assert seen >= 8
