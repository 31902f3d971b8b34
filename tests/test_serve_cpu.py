"""CPU (no GPU needed): the serving operators' C structs as paia_gemv.serve packs them, their refusals on the host (code
-2 before any device is touched), the checks of the tensor wrappers (ValueError), and a replay of the attention's division
of work and of the adapters' finding of their rows."""
import random
import re
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
PTR = 0x10000


@pytest.fixture(scope="module")
def L(lib_path):
    from paia_gemv import loader
    return loader.GemvLib(lib_path)


def fields(name):
    """The field names of a struct of the header, in order, and their kinds (P pointer, q, i, f)."""
    txt = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "paia_gemv.h").read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, txt, flags=re.S).group(1)
    out = []
    for decl in body.split(";"):
        decl = decl.strip()
        if not decl:
            continue
        kind = "P" if "*" in decl else "q" if decl.startswith("long long") else "f" if decl.startswith("float") else "i"
        names = re.sub(r"^(const )?(void|int|float|double|long long)\b", "", decl)
        out += [(n.strip(" *"), kind) for n in names.split(",")]
    return out


def packed(name, fmt, good, **change):
    values = dict(good)
    values.update(change)
    names = fields(name)
    assert {n for n, _ in names} == set(values)
    return fmt.pack(*[values[n] for n, _ in names])


ATTN = dict(q=PTR, k=PTR, v=PTR, page_table=PTR, lens=PTR, k_scale=0, v_scale=0, out=PTR, lse=0, workspace=PTR,
            q_batch=1024, q_head=128, out_batch=1024, out_head=128, lse_batch=8, table_batch=4, k_page=4096, k_token=256,
            k_head=128, v_page=4096, v_token=256, v_head=128, batch=2, heads=8, kv_heads=2, head_dim=128, cache=0,
            num_pages=9, page_size=16, max_pages=4, window=0, scale=0.1)
ROPE = dict(qkv=PTR, pos=PTR, seq=0, inv_freq=PTR, q_norm=0, k_norm=0, page_table=PTR, k_scale=0, v_scale=0, q_out=PTR,
            k_out=0, k=PTR, v=PTR, qkv_token=1536, q_token=1024, q_head=128, ko_token=0, ko_head=0, table_seq=4,
            k_page=4096, k_row=256, k_head=128, v_page=4096, v_row=256, v_head=128, tokens=3, sequences=3, heads=8,
            kv_heads=2, head_dim=128, rot=128, interleaved=0, cache=0, num_pages=9, page_size=16, max_pages=4, eps=1e-6)
LORA = dict(x=PTR, a=PTR, b=PTR, adapter=PTR, ranks=0, scaling=0, base=0, out=2 * PTR, x_row=64, base_row=0, out_row=64,
            a_adapter=512, a_row=64, b_adapter=512, b_row=8, M=3, N=64, K=64, rank=8, adapters=2)


def test_structs_match_the_header(tmp_path):
    from paia_gemv import serve
    names = {"paia_gemv_attn": serve.ATTN, "paia_gemv_rope_cache": serve.ROPE_CACHE, "paia_gemv_lora_args": serve.LORA}
    for n, fmt in names.items():
        kinds = "".join(k for _, k in fields(n))
        spelled = "".join(k * int(c or 1) for c, k in re.findall(r"(\d*)([Pqif])", fmt.format))
        assert kinds == spelled, n
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "paia_gemv.h"\nint main(void) { printf("'
                   + " ".join(["%zu"] * 3) + '", ' + ", ".join(f"sizeof({n})" for n in names) + "); return 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [f.size for f in names.values()]


@pytest.mark.parametrize("change", [
    dict(heads=7), dict(heads=0), dict(kv_heads=0), dict(head_dim=80), dict(head_dim=512), dict(batch=-1), dict(cache=2),
    dict(cache=-1), dict(page_size=0), dict(max_pages=-1), dict(num_pages=0), dict(window=-1), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=0), dict(k=0), dict(v=0),
    dict(page_table=0), dict(lens=0), dict(out=0), dict(workspace=0), dict(q=PTR + 2), dict(k=PTR + 8), dict(v=PTR + 8),
    dict(workspace=PTR + 4), dict(out=PTR + 4), dict(lse=PTR + 2), dict(lens=PTR + 2), dict(page_table=PTR + 1),
    dict(q_batch=1020), dict(q_head=130), dict(out_head=127), dict(k_token=260), dict(v_page=4100), dict(k_head=129),
    dict(k_scale=PTR), dict(v_scale=PTR), dict(cache=1, k_token=264), dict(cache=1, k_scale=PTR + 1),
    dict(page_size=65536, max_pages=65536), dict(batch=1 << 20, max_pages=1 << 16), dict(out_head=0), dict(out_batch=0),
    dict(lse=PTR, lse_batch=0)])
def test_attention_refusals(L, change):
    from paia_gemv import serve
    assert L._lib.paia_gemv_paged_attn(packed("paia_gemv_attn", serve.ATTN, ATTN, **change), None) == -2


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(heads=0), dict(kv_heads=0), dict(head_dim=24), dict(head_dim=272), dict(head_dim=0), dict(rot=8),
    dict(rot=144), dict(rot=-16), dict(cache=3), dict(eps=-1.0), dict(eps=float("nan")), dict(qkv=0), dict(pos=0),
    dict(q_out=0), dict(inv_freq=0), dict(k=0), dict(v=0), dict(k=0, v=0), dict(page_table=0), dict(sequences=0),
    dict(num_pages=0), dict(page_size=0), dict(max_pages=0), dict(k_scale=PTR), dict(qkv=PTR + 2), dict(q_out=PTR + 8),
    dict(k=PTR + 8), dict(k_out=PTR + 4), dict(q_norm=PTR + 4), dict(inv_freq=PTR + 4), dict(pos=PTR + 2),
    dict(qkv_token=1537), dict(q_token=4), dict(q_head=12), dict(ko_token=4), dict(k_row=260), dict(v_head=3),
    dict(cache=1, v_row=264), dict(q_head=0), dict(q_token=0), dict(k_head=0), dict(v_row=0), dict(k_page=0),
    dict(k_out=PTR, ko_head=0, ko_token=256), dict(k_out=PTR, ko_head=128, ko_token=0)])
def test_rope_refusals(L, change):
    from paia_gemv import serve
    args = packed("paia_gemv_rope_cache", serve.ROPE_CACHE, ROPE, **change)
    assert L._lib.paia_gemv_qkv_rope_cache(args, None) == -2


@pytest.mark.parametrize("change", [
    dict(M=-1), dict(N=0), dict(N=60), dict(K=0), dict(K=4), dict(K=60), dict(rank=0), dict(rank=12), dict(rank=264),
    dict(adapters=0), dict(adapters=8193), dict(x=0), dict(a=0), dict(b=0), dict(adapter=0), dict(out=0), dict(x=PTR + 8),
    dict(a=PTR + 2), dict(b=PTR + 4), dict(base=PTR + 8), dict(out=PTR + 8), dict(adapter=PTR + 2), dict(ranks=PTR + 1),
    dict(scaling=PTR + 2), dict(x_row=65), dict(base_row=4), dict(out_row=68), dict(a_adapter=4), dict(a_row=66),
    dict(b_adapter=2), dict(b_row=12), dict(out_row=0), dict(out=PTR), dict(M=(1 << 30) + 1)])
def test_lora_refusals(L, change):
    from paia_gemv import serve
    assert L._lib.paia_gemv_lora(packed("paia_gemv_lora_args", serve.LORA, LORA, **change), None) == -2


def test_nothing_to_do_and_null(L):
    from paia_gemv import serve
    lib = L._lib
    assert lib.paia_gemv_paged_attn(packed("paia_gemv_attn", serve.ATTN, ATTN, batch=0), None) == 0
    assert lib.paia_gemv_qkv_rope_cache(packed("paia_gemv_rope_cache", serve.ROPE_CACHE, ROPE, tokens=0), None) == 0
    assert lib.paia_gemv_lora(packed("paia_gemv_lora_args", serve.LORA, LORA, M=0), None) == 0
    assert lib.paia_gemv_paged_attn(None, None) == lib.paia_gemv_qkv_rope_cache(None, None) == -2
    assert lib.paia_gemv_lora(None, None) == -2
    assert lib.paia_gemv_paged_attn_workspace(8, 3, 128) == lib.paia_gemv_paged_attn_workspace(8, 2, 100) == 0
    with pytest.raises(RuntimeError):
        L.paged_attn_workspace(8, 3, 128)
    with pytest.raises(RuntimeError):
        L._check(L.lora(packed("paia_gemv_lora_args", serve.LORA, LORA, rank=12), 0), "paia_gemv_lora")
    assert L.paged_attn_workspace(32, 8, 128) < L.paged_attn_workspace(64, 8, 128) <= 16 << 20


def test_wrappers_refuse_tensors_off_the_device(L):
    from paia_gemv import serve
    bf, i32 = torch.bfloat16, torch.int32
    q, pool = torch.zeros(1, 4, 64, dtype=bf), torch.zeros(2, 16, 2, 64, dtype=bf)
    one = torch.zeros(1, dtype=i32)
    with pytest.raises(ValueError, match="current CUDA device"):
        serve.paged_attention(L, q, pool, pool, one.view(1, 1), one, q,
                              serve.AttentionWorkspace(torch.zeros(1 << 20, dtype=torch.uint8), 4, 2, 64))
    with pytest.raises(ValueError, match="current CUDA device"):
        serve.qkv_rope_cache(L, torch.zeros(1, 8 * 64, dtype=bf), one, torch.ones(32, dtype=torch.float64), q, pool, pool,
                             one.view(1, 1))
    with pytest.raises(ValueError, match="current CUDA device"):
        serve.lora(L, torch.zeros(1, 64, dtype=bf), torch.zeros(1, 8, 64, dtype=bf), torch.zeros(1, 64, 8, dtype=bf), one,
                   torch.zeros(1, 64, dtype=bf))


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on CUDA device 0: the wrappers' checks run, nothing is launched."""
    def get_device(self):
        return 0


def on(t):
    return t.as_subclass(OnDevice)


class Recorder:
    """Stands in for the library: takes the packed struct."""
    paged_attn_entry = qkv_rope_cache_entry = lora_entry = device_entry = 0

    def __init__(self):
        self.calls = []

    def paged_attn(self, args, stream):
        self.calls.append(args)
        return 0

    qkv_rope_cache = lora = paged_attn


def test_wrapper_raises_return_codes(monkeypatch, L):
    from paia_gemv import serve
    monkeypatch.setattr(serve, "_current_device", lambda: 0)
    z = lambda *s, dtype=torch.bfloat16: on(torch.zeros(*s, dtype=dtype))   # noqa: E731
    with pytest.raises(RuntimeError, match="paia_gemv_lora failed with code -2"):      # rank 12 is no multiple of 8
        serve.lora(L, z(3, 64), z(2, 12, 64), z(2, 40, 12), z(3, dtype=torch.int32), z(3, 40), stream=0)


def test_wrapper_checks(monkeypatch):
    """Every tensor of a call is checked for its type, shape, layout and device before the library sees it."""
    from paia_gemv import serve
    monkeypatch.setattr(serve, "_current_device", lambda: 0)
    monkeypatch.setattr(serve, "_raw_stream", lambda d: 0)
    bf, i32, rec = torch.bfloat16, torch.int32, Recorder()
    z = lambda *s, dtype=bf: on(torch.zeros(*s, dtype=dtype))   # noqa: E731
    good = dict(q=z(3, 4, 64), k_pages=z(5, 16, 2, 64), v_pages=z(5, 16, 2, 64), page_table=z(3, 6, dtype=i32),
                lens=z(3, dtype=i32), out=z(3, 4, 64), workspace=serve.AttentionWorkspace(z(64, dtype=torch.uint8), 4, 2, 64))
    serve.paged_attention(rec, **good)
    hnd = z(5, 2, 16, 64).transpose(1, 2)
    serve.paged_attention(rec, **dict(good, k_pages=hnd, v_pages=hnd), lse=z(3, 4, dtype=torch.float32), window=5)
    vals = serve.ATTN.unpack(rec.calls[1])
    names = [n for n, _ in fields("paia_gemv_attn")]
    got = dict(zip(names, vals))
    assert (got["batch"], got["heads"], got["kv_heads"], got["head_dim"]) == (3, 4, 2, 64)
    assert (got["num_pages"], got["page_size"], got["max_pages"], got["window"]) == (5, 16, 6, 5)
    assert (got["k_page"], got["k_token"], got["k_head"]) == (2 * 16 * 64, 64, 16 * 64)
    assert abs(got["scale"] - 0.125) < 1e-9 and got["lse"] and not got["k_scale"]
    f32 = torch.float32
    for bad in (dict(q=z(3, 4, 64, dtype=f32)), dict(q=z(3, 5, 64)), dict(q=z(4, 64)), dict(q=z(3, 64, 4).transpose(1, 2)),
                dict(k_pages=z(5, 16, 2, 128)), dict(k_pages=z(5, 16, 128)), dict(v_pages=z(4, 16, 2, 64)),
                dict(v_pages=z(5, 16, 2, 64, dtype=torch.float8_e4m3fn)), dict(k_pages=z(5, 16, 2, 64, dtype=f32)),
                dict(page_table=z(2, 6, dtype=i32)), dict(page_table=z(3, 6, dtype=torch.int64)),
                dict(page_table=z(18, dtype=i32)), dict(lens=z(2, dtype=i32)), dict(lens=z(3, dtype=torch.int64)),
                dict(lens=z(6, dtype=i32)[::2]), dict(out=z(3, 4, 32)), dict(out=z(3, 4, 64, dtype=f32)),
                dict(workspace=serve.AttentionWorkspace(z(64, dtype=torch.uint8), 4, 4, 64)),
                dict(workspace=serve.AttentionWorkspace(torch.zeros(64, dtype=torch.uint8), 4, 2, 64)), dict(k_scale=z(2, dtype=f32)),
                dict(lse=z(3, 5, dtype=f32)), dict(lse=z(3, 4)), dict(lens=torch.zeros(3, dtype=i32)),
                dict(v_pages=torch.zeros(5, 16, 2, 64, dtype=bf))):
        with pytest.raises(ValueError):
            serve.paged_attention(rec, **dict(good, **bad))
    good = dict(qkv=z(3, 8 * 64), positions=z(3, dtype=i32), inv_freq=z(32, dtype=torch.float64), q_out=z(3, 4, 64),
                k_pages=z(5, 16, 2, 64), v_pages=z(5, 16, 2, 64), page_table=z(3, 6, dtype=i32))
    serve.qkv_rope_cache(rec, **good)
    serve.qkv_rope_cache(rec, **dict(good, page_table=z(1, 6, dtype=i32)), seq=z(3, dtype=i32))
    none = dict(good, k_pages=None, v_pages=None, page_table=None)
    serve.qkv_rope_cache(rec, **none, k_out=z(3, 2, 64), kv_heads=2)
    for bad in (dict(qkv=z(3, 7 * 64)), dict(qkv=z(2, 8 * 64)), dict(positions=z(2, dtype=i32)),
                dict(positions=z(3, dtype=torch.int64)), dict(inv_freq=z(32, dtype=f32)), dict(inv_freq=z(4, 8, dtype=torch.float64)),
                dict(q_out=z(3, 256)), dict(page_table=z(2, 6, dtype=i32)), dict(seq=z(2, dtype=i32)),
                dict(q_norm=z(64)), dict(k_norm=z(32, dtype=f32)), dict(k_out=z(3, 1, 64)), dict(v_scale=z(2, dtype=f32)),
                dict(v_pages=z(5, 16, 2, 64).transpose(0, 3))):
        with pytest.raises(ValueError):
            serve.qkv_rope_cache(rec, **dict(good, **bad))
    for bad in (none, dict(none, k_out=z(3, 2, 64)), dict(none, kv_heads=2), dict(good, k_pages=None)):
        with pytest.raises(ValueError):
            serve.qkv_rope_cache(rec, **bad)
    good = dict(x=z(3, 64), a=z(2, 8, 64), b=z(2, 40, 8), adapter=z(3, dtype=i32), out=z(3, 40))
    serve.lora(rec, **good)
    for bad in (dict(x=z(3, 32)), dict(x=z(64)), dict(a=z(8, 64)), dict(a=z(2, 8, 64, dtype=f32)), dict(b=z(2, 40, 16)),
                dict(b=z(1, 40, 8)), dict(adapter=z(2, dtype=i32)), dict(adapter=z(3, dtype=torch.int64)),
                dict(out=z(3, 48)), dict(base=z(2, 40)), dict(base=z(3, 40, dtype=f32)), dict(scaling=z(3, dtype=f32)),
                dict(scaling=z(2)), dict(ranks=z(2, dtype=f32)), dict(out=z(40, 3).t())):
        with pytest.raises(ValueError):
            serve.lora(rec, **dict(good, **bad))


def attention_division(lens, units, pos, grid, warps, cost, window):
    """What each CTA of serve_attn.cu works on: {cta: [(sequence, unit, first tile, tiles of the part, tiles of the unit,
    c0, c1)]}, as the kernel finds it."""
    def tiles(n):
        start = n - window if window and n > window else 0
        return max(1, (n + pos - 1) // pos - start // pos)

    each = [tiles(n) + cost for n in lens]
    total = sum(each) * units
    per = max(-(-total // grid), warps)
    out = {}
    for cta in range(grid):
        if per * cta >= total:
            continue
        t0 = per * cta
        t1 = t0 + min(total - t0, per)
        b, before = 0, 0
        while t0 >= (before + each[b]) * units:
            before += each[b]
            b += 1
        w0 = before * units
        u, tile = divmod(t0 - w0, each[b])
        n = each[b] - cost

        def following(b, u, w0):
            if u + 1 < units:
                return b, u + 1, w0
            return b + 1, 0, w0 + each[b] * units

        if tile >= n:                                           # behind its unit's tiles
            b, u, w0 = following(b, u, w0)
            tile = 0
            if b == len(lens) or w0 + u * each[b] >= t1:
                continue
        while True:
            n, place = each[b] - cost, w0 + u * each[b]
            part = min(n, t1 - place) - tile
            assert part > 0
            out.setdefault(cta, []).append((b, u, tile, part, n, place // per, (place + n - 1) // per))
            if place + each[b] >= t1:
                break
            b, u, w0 = following(b, u, w0)
            tile = 0
    return out


def test_attention_division_covers_every_tile_once():
    """Every tile of every unit belongs to one CTA; a unit in parts is counted in by exactly the CTAs c0 .. c1, the counter
    of c0 and each CTA's two slots of the workspace serve one unit each."""
    src = (ROOT / "paia-project_b200" / "csrc" / "serve_attn.cu").read_text()
    costs = dict(zip((4, 2), map(int, re.search(r"unit_cost.*W == 4 \? (\d+) : (\d+);", src).groups())))
    rng = random.Random(4)
    for trial in range(300):
        lens = [rng.choice([0, 1, rng.randrange(40), rng.randrange(3000)]) for _ in range(rng.choice([1, 2, 7, 40, 90]))]
        units, pos, grid = rng.choice([1, 2, 8, 13]), rng.choice([16, 32]), rng.choice([1, 5, 148, 296])
        window = rng.choice([0, 0, 1, 100])
        warps = rng.choice([4, 2])
        work = attention_division(lens, units, pos, grid, warps, costs[warps], window)
        seen, arrivals, counters, slots = {}, {}, {}, {}
        for cta, parts in work.items():
            for b, u, tile, part, n, c0, c1 in parts:
                for i in range(tile, tile + part):
                    assert seen.setdefault((b, u, i), cta) == cta
                if part < n:
                    arrivals.setdefault((b, u, c0, c1), []).append(cta)
                    assert counters.setdefault(c0, (b, u)) == (b, u)
                    slot = (cta, 1 if tile == 0 else 0)
                    assert slots.setdefault(slot, (b, u)) == (b, u)
                    assert slot[1] == (1 if cta == c0 else 0)   # where the join looks for it
                else:
                    assert c0 == c1 == cta or c0 <= cta <= c1
        for b, n in enumerate(lens):
            start = n - window if window and n > window else 0
            count = max(1, (n + pos - 1) // pos - start // pos)
            for u in range(units):
                assert all((b, u, i) in seen for i in range(count)) and (b, u, count) not in seen
        for (b, u, c0, c1), ctas in arrivals.items():
            assert sorted(ctas) == list(range(c0, c1 + 1)), (lens, b, u)


def test_adapter_items_cover_every_row_once():
    """The number of clusters that the host launches is enough for any assignment of rows, and the items of up to 16 rows
    (by order of the row that begins them, or by adapter beyond 256 rows) hold every row once."""
    rng = random.Random(5)
    for trial in range(200):
        adapters = rng.choice([1, 2, 5, 60, 500])
        m = rng.choice([1, 3, 16, 17, 100, 256, 257, 700])
        ids = [rng.choice([rng.randrange(adapters), adapters, 0]) for _ in range(m)]
        kinds = min(m, adapters + 1)
        items = (m + 15 * kinds) // 16
        at = [sum(ids[j] == ids[i] for j in range(i)) for i in range(m)]
        if m <= 256:
            begins = [i for i in range(m) if at[i] % 16 == 0]
            rows = [[i for i in range(m) if ids[i] == ids[s] and at[s] <= at[i] < at[s] + 16] for s in begins]
        else:
            rows = []
            for a in range(adapters + 1):
                mine = [i for i in range(m) if ids[i] == a]
                rows += [mine[k:k + 16] for k in range(0, len(mine), 16)]
        assert len(rows) <= items and sorted(i for r in rows for i in r) == list(range(m))


def adapter_run(counts, key, m, item, end):
    """(adapter, rows) of each item of a CTA's run [item, end), as the kernel searches for them 1024 rows at a time."""
    scan, out = (-1, 0, 0), []
    while item < end:
        before, found = 0, None
        for a, c in enumerate(counts):
            n = (c + 15) // 16
            if before <= item < before + n:
                found = (a, (item - before) * 16, min(16, c - (item - before) * 16))
            before += n
        if found is None:
            break
        a, skip, want = found
        m0, seen = scan[1:] if scan[0] == a else (0, 0)
        rows = {}
        while seen < skip + want:
            assert m0 < m
            mine = [r for r in range(m0, min(m0 + 1024, m)) if key[r] == a]
            rows.update({seen + i - skip: r for i, r in enumerate(mine) if skip <= seen + i < skip + want})
            scan = (a, m0, seen)
            seen, m0 = seen + len(mine), m0 + 1024
        out.append((a, [rows[i] for i in range(want)]))
        item += 1
    return out


def test_adapter_runs_cover_every_row_once():
    """More than 256 rows: the CTAs' runs of items hold every row once, under its adapter and in order, whatever the grid."""
    rng = random.Random(6)
    for trial in range(40):
        m, adapters, grid = rng.choice([257, 1024, 1025, 4000]), rng.choice([1, 2, 7, 300]), rng.choice([1, 7, 64, 296])
        key = [rng.randrange(adapters + 1) if trial % 2 else min(r * r % (adapters + 3), adapters) for r in range(m)]
        counts = [key.count(a) for a in range(adapters + 1)]
        items = sum((c + 15) // 16 for c in counts)
        got = []
        for cta in range(grid):
            got += adapter_run(counts, key, m, items * cta // grid, items * (cta + 1) // grid)
        assert len(got) == items and sorted(r for _, rows in got for r in rows) == list(range(m))
        for a, rows in got:
            assert rows == sorted(rows) and all(key[r] == a for r in rows)


def test_attention_clusters_cover_every_tile_once():
    """A small call's CTAs take neighbouring runs of their unit's tiles; the first has one at least."""
    for log2 in (1, 2, 3):
        c = 1 << log2
        for n in range(1, 300):
            runs = [((n * r + c - 1) >> log2, (n * (r + 1) + c - 1) >> log2) for r in range(c)]
            assert runs[0][0] == 0 and runs[0][1] > 0 and runs[-1][1] == n
            assert all(x[1] == y[0] for x, y in zip(runs, runs[1:]))
