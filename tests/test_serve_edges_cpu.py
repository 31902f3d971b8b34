"""CPU (no GPU needed): refusals and host-side decisions of the serving operators that the calls of test_serve_cpu.py do not
reach."""
import platform
import random
import re
import shutil
import sysconfig
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def L(lib_path):
    from paia_gemv import loader
    return loader.GemvLib(lib_path)


class OnCuda(torch.Tensor):
    """A CPU tensor that says it is on CUDA device 0: host-side checks run, nothing is launched."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (32, 8, 128), (64, 2, 256), (40, 2, 96)])
def test_workspace_over_a_buffer(L, heads, kv, hd):
    """A workspace over a caller's own buffer holds what the kernel may write, or is refused."""
    from paia_gemv import serve
    need = L.paged_attn_workspace(heads, kv, hd)
    buf = lambda n, dtype=torch.uint8: torch.zeros(n, dtype=dtype).as_subclass(OnCuda)   # noqa: E731
    whole = buf(need + 16)
    at = -whole.data_ptr() % 16
    ws = serve.AttentionWorkspace(whole[at:at + need], heads, kv, hd, L)
    assert ws.ptr % 16 == 0 and ws.sizes == (0, heads, kv, hd)
    for bad in (whole[at:at + need - 1], buf(64), buf(0), whole[at + 1:at + 1 + need], buf(2 * need + 32)[::2],
                buf(need, torch.int8), buf(need, torch.float32)):
        with pytest.raises(ValueError, match="buffer must be"):
            serve.AttentionWorkspace(bad, heads, kv, hd, L)
    with pytest.raises(RuntimeError):                            # heads that the attention does not take
        serve.AttentionWorkspace(whole, heads + 1, kv, hd, L)


def test_extension_of_another_interpreter_is_not_loaded(L, monkeypatch, tmp_path):
    """The extension's name carries the interpreter that it was built for, and only this one's is loaded."""
    from paia_gemv import serve
    if serve._bind is None:
        pytest.skip("the extension is not built")
    assert serve._bind.__file__.endswith("_paia_serve" + sysconfig.get_config_var("EXT_SUFFIX"))
    monkeypatch.setattr(serve, "_PKG_ROOT", tmp_path)
    at = tmp_path / "build" / platform.machine()
    at.mkdir(parents=True)
    for name in ("_paia_serve.so", "_paia_serve.cpython-31-x86_64-linux-gnu.so"):
        shutil.copy(serve._bind.__file__, at / name)
    assert serve._load_bind() is None


def scans(each, units, t0):
    """(sequence, places before it) of place t0, as every warp of the attention finds it: lane i adds up the i-th share of
    the sequences, one scan over the lanes finds the share, scans of 32 of its sequences at a time the sequence."""
    batch = len(each)
    share = (batch + 31) // 32
    mine = [sum(each[min(i * share, batch):min(min(i * share, batch) + share, batch)]) for i in range(32)]
    inc = [sum(mine[:i + 1]) for i in range(32)]
    lane = next(i for i in range(32) if t0 < inc[i] * units)
    before, at = inc[lane] - mine[lane], lane * share
    if share > 1:
        end = min(at + share, batch)
        while True:
            n = [each[at + i] if at + i < end else 0 for i in range(32)]
            inc = [sum(n[:i + 1]) for i in range(32)]
            hits = [i for i in range(32) if t0 < (before + inc[i]) * units]
            if hits or at + 32 >= end:
                i = hits[0] if hits else 31
                at, before = at + i, before + inc[i] - n[i]
                break
            before, at = before + inc[31], at + 32
    return at, before


@pytest.mark.parametrize("batch", [1, 31, 32, 33, 64, 65, 700, 1023, 1024, 1025, 1056, 1057, 1100, 2048, 2049, 2100, 3300, 5000])
def test_attention_start_is_found_at_any_batch(batch):
    """Beyond 1024 sequences a lane's share is more than 32: the scans go on over it."""
    rng = random.Random(batch)
    for units in (1, 3, 8):
        each = [rng.choice([7, 8, 1 + 14, rng.randrange(7, 400)]) for _ in range(batch)]
        starts, place = [], 0
        for n in each:
            starts.append(place)
            place += n * units
        per = max(-(-place // rng.choice([148, 296, 592])), 4)
        for t0 in sorted({t for t in range(0, place, per)} | {0, place - 1} | {rng.choice(starts) for _ in range(20)}
                         | {max(rng.choice(starts) - 1, 0) for _ in range(20)}):
            b, before = scans(each, units, t0)
            assert before * units == starts[b] <= t0 < starts[b] + each[b] * units


def test_value_brackets_find_every_border():
    """What an e4m3 cache stores of v: the fp32 quotients of v less and plus a margin, by the reciprocal of the scale. Where
    both round to one e4m3 value that is the value nearest to the exact quotient, for every bf16 mantissa and every scale
    within eight fp32 steps of putting it on a border (beyond them the margin is not needed)."""
    src = (ROOT / "paia-project_b200" / "csrc" / "serve_rope.cu").read_text()
    margin = torch.tensor(float(re.search(r"fabsf\(l\[i\]\) \* ([\d.e-]+)f;", src).group(1)))

    def nearest(x):                                              # of a binade from 1 on, or of the subnormal values
        step = torch.where(x >= 0.25, 2.0 ** -3, 2.0 ** -9).double()
        return torch.round(x.double() / step) * step

    normal = (2 * torch.arange(8, 16).double() + 1) / 16
    for m, step in ((normal, 2.0 ** -3), ((2 * torch.arange(8).double() + 1) * 2.0 ** -10, 2.0 ** -9)):
        v = (1 + torch.arange(128) / 128).float()[:, None, None].expand(128, 8, 17)
        s = (v[:, :, 0].double() / m).float()
        s = (s[..., None].view(torch.int32) + torch.arange(-8, 9, dtype=torch.int32)).view(torch.float32)
        off, inv = v * margin, 1 / s
        lo, hi = nearest((v - off) * inv), nearest((v + off) * inv)
        d = v.double() - m[None, :, None] * s.double()          # exact: 5 bits by 24
        below = (m - step / 2)[None, :, None].expand_as(d)
        tie = torch.where(torch.round(below / step) % 2 == 0, below, below + step)
        want = torch.where(d < 0, below, torch.where(d > 0, below + step, tie))
        assert ((lo == hi) <= (lo == want)).all() and ((lo <= want) & (want <= hi)).all()
        assert (lo != hi).any() and (lo == hi).any()


def test_registers_and_spills():
    """ptxas's report of the serving kernels: two CTAs of the attention fit an SM wherever they are launched so, and only
    known instances spill, none by more than it does: head_dim 256 (its sums fill the registers), 16 heads beside an e4m3
    cache at head_dim 128, and the adapters' search among more than 256 rows (a few bytes)."""
    from test_compile_report import load_reports
    rows = [r for r in load_reports() if r["file"].startswith("serve_")]
    assert len(rows) >= 36 + 2 + 2
    seen = 0
    for r in rows:
        spills = r["spill_st"] + r["spill_ld"]
        m = re.search(r"paged_attn_kernelILi(\d+)ELi(\d)ELi(\d+)ELi(\d)ELi(\d)ELi(\d)ELb(\d)E", r["fn"])
        if m:
            hd, fmt, heads, warps, _, ctas, _ = map(int, m.groups())
            seen += 1
            assert r["regs"] * warps * 32 * ctas <= 65536, r
            known = 700 if hd == 256 else 300 if (hd, fmt, heads) == (128, 1, 16) else 0
            assert spills <= known and r["stack"] <= known, r
        elif "lora_kernel" in r["fn"]:
            assert spills <= 64 and r["regs"] * 512 <= 65536, r
        else:
            assert "qkv_rope_kernel" in r["fn"] and spills == 0 and r["stack"] <= 16, r   # (a frame for the settled bytes)
    assert seen >= 36


@pytest.mark.parametrize("change", [
    dict(batch=1 << 19, heads=4096, kv_heads=4096, max_pages=1, page_size=16), dict(max_pages=1, page_size=0x7FFFFF01),
    dict(batch=1 << 28, heads=2, kv_heads=1, max_pages=0), dict(batch=1 << 24, heads=512, kv_heads=1, max_pages=0)])
def test_attention_size_limits(L, change):
    """The limits that the header gives for positions and places: short tables count 16 places per unit."""
    import test_serve_cpu as T
    from paia_gemv import serve
    a = dict(T.ATTN, q_batch=0, **change)
    places = a["batch"] * a["kv_heads"] * -(-(a["heads"] // a["kv_heads"]) // 16) * (a["max_pages"] * a["page_size"] // 16 + 16)
    assert a["max_pages"] * a["page_size"] > 2 ** 31 - 256 or places > 2 ** 32 - 2 ** 20
    assert L._lib.paia_gemv_paged_attn(T.packed("paia_gemv_attn", serve.ATTN, a), None) == -2
    if a["batch"] > 2:                                           # its own size alone is what is refused
        assert L._lib.paia_gemv_paged_attn(T.packed("paia_gemv_attn", serve.ATTN, dict(a, batch=0)), None) == 0


def test_strides_of_one_do_not_count(monkeypatch):
    """Python's route: the stride of a dimension of one may be anything (a row of a wider buffer, one head of many) and the
    struct holds 0 for it, as the extension's route has it."""
    import test_serve_cpu as T
    from paia_gemv import serve
    monkeypatch.setattr(serve, "_bind", None)
    monkeypatch.setattr(serve, "_current_device", lambda: 0)
    monkeypatch.setattr(serve, "_raw_stream", lambda d: 0)
    rec = T.Recorder()

    def odd(*shape, dtype=torch.bfloat16):
        """Zeros of this shape whose dimensions of one have the stride 13."""
        t = torch.zeros(shape, dtype=dtype)
        return T.on(t.as_strided(shape, [13 if n == 1 else s for n, s in zip(shape, t.stride())]))

    def packed(name, fmt):
        return dict(zip([n for n, _ in T.fields(name)], fmt.unpack(rec.calls[-1])))
    i32, f32 = torch.int32, torch.float32
    serve.paged_attention(rec, odd(1, 1, 64), odd(1, 1, 1, 64), odd(1, 1, 1, 64), odd(1, 6, dtype=i32), odd(1, dtype=i32),
                          odd(1, 1, 64), serve.AttentionWorkspace(odd(64, dtype=torch.uint8), 1, 1, 64),
                          lse=odd(1, 1, dtype=f32))
    got = packed("paia_gemv_attn", serve.ATTN)
    assert not any(v for n, v in got.items() if n.split("_")[0] in "qkv" and n.split("_")[-1] in ("batch", "head", "page", "token"))
    assert got["out_batch"] == got["out_head"] == got["lse_batch"] == got["table_batch"] == 0
    serve.qkv_rope_cache(rec, odd(1, 3 * 64), odd(1, dtype=i32), odd(32, dtype=torch.float64), odd(1, 1, 64), odd(1, 1, 1, 64),
                         odd(1, 1, 1, 64), odd(1, 1, dtype=i32), k_out=odd(1, 1, 64))
    got = packed("paia_gemv_rope_cache", serve.ROPE_CACHE)
    assert not any(got[n] for n in ("qkv_token", "q_token", "q_head", "ko_token", "ko_head", "table_seq", "k_page", "k_row",
                                    "k_head", "v_page", "v_row", "v_head"))
    serve.lora(rec, odd(1, 64), odd(1, 8, 64), odd(1, 40, 8), odd(1, dtype=i32), odd(1, 40), base=odd(1, 40))
    got = packed("paia_gemv_lora_args", serve.LORA)
    assert not any(got[n] for n in ("x_row", "base_row", "out_row", "a_adapter", "b_adapter")) and got["a_row"] == 64
