"""Serving operators on torch tensors: what a batched decode step does between its GEMVs (include/paia_gemv.h has the
definitions). Each call checks its tensors, packs the C struct and launches on torch's current stream (or `stream`);
outputs are written in place, nothing is allocated and nothing synchronises, so every call is CUDA-graph capturable.

    qkv_rope_cache   per-head norm, rotary positions and cache write of a fused QKV projection's rows
    paged_attention  attention of one new token per sequence over the paged cache
    lora             the low-rank adapters of many requests, added to a shared projection
    route            each token's experts and their weights, and the tokens grouped by expert (a `routing`)
    expert_matmul    the products of each group with its expert's weights
    block_norm       a block's (weighted) output, normed, gated and added to the residual, and the norm before the next one

Caches are a pair of tensors [num_pages, page_size, kv_heads, head_dim] (bf16, or float8_e4m3fn with a fp32 scale per
kv head), in any layout whose head_dim is contiguous: a [num_pages, kv_heads, page_size, head_dim] pool is passed as
`pool.transpose(1, 2)`. Page tables are int32 [sequences, max_pages]. Tensors live on the current CUDA device.
"""
import importlib.util
import platform
import struct
import sysconfig

import torch

from .loader import _PKG_ROOT, load_lib

# the C structs, field by field (native alignment): include/paia_gemv.h
ATTN = struct.Struct("10P 12q 9i f")
ROPE_CACHE = struct.Struct("13P 12q 11i f")
LORA = struct.Struct("8P 7q 5i 4x")
ROUTE = struct.Struct("9P q 6i f 4x")
EXPERTS = struct.Struct("7P 5q 8i")
BLOCK_NORM = struct.Struct("9P 7q 5i 2f i")

def _load_bind():
    """The extension that checks and makes these calls in C (csrc/serve_bind.cpp), or None: without it, and for every
    call that it does not find exactly as it should be, the code below checks, calls and raises. One built for another
    interpreter (its name says which) is not looked at."""
    path = _PKG_ROOT / "build" / platform.machine() / ("_paia_serve" + sysconfig.get_config_var("EXT_SUFFIX"))
    api = getattr(torch.Tensor, "__dlpack_c_exchange_api__", None)
    if api is None or not path.exists():
        return None
    try:
        spec = importlib.util.spec_from_file_location("_paia_serve", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    except ImportError:
        return None
    return mod if mod.init(torch.Tensor, api) else None


_bind = _load_bind()

# torch.cuda.current_device() and current_stream() without their Python layers (absent from CPU builds of torch)
_current_device = getattr(torch._C, "_cuda_getDevice", lambda: -1)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0)
_pack_attn, _pack_rope, _pack_lora = ATTN.pack, ROPE_CACHE.pack, LORA.pack
_pack_route, _pack_experts, _pack_norm = ROUTE.pack, EXPERTS.pack, BLOCK_NORM.pack
_BF16, _F32, _F64, _I32, _E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.float8_e4m3fn
_U8 = torch.uint8


def _bad(name, t, what):
    raise ValueError(f"{name} must be {what} on the current CUDA device, got "
                     + (f"{t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}"
                        if isinstance(t, torch.Tensor) else repr(t)))


# The checks are written out call by call (a decode step makes them on its critical path): a tensor's shape, type,
# device and contiguous last dimension, then its pointer and strides into the struct.

def _flat(name, t, dtype, shape, dev):
    """The pointer of a contiguous tensor of this shape; 0 for None."""
    if t is None:
        return 0
    if t.shape != shape or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        _bad(name, t, f"contiguous {dtype} {shape}")
    return t.data_ptr()


def _strides(t):
    """The strides of a tensor, 0 along a dimension of one: never used, and free to be anything in torch."""
    shape, strides = t.shape, t.stride()
    return tuple([0 if n == 1 else s for n, s in zip(shape, strides)]) if 1 in shape else strides


def _device(t, name):
    dev = t.get_device()
    if dev < 0 or dev != _current_device():
        raise ValueError(f"{name} is on {t.device}: the operators run on the current CUDA device")
    return dev


def _pools(k, v, kv_heads, head_dim, k_scale, v_scale, dev):
    """(cache code, pool shape, strides of k, of v) of a cache's two pools."""
    shape, dtype, ks, vs = k.shape, k.dtype, _strides(k), _strides(v)
    if len(shape) != 4 or shape[2] != kv_heads or shape[3] != head_dim:
        _bad("k_pages", k, f"[num_pages, page_size, {kv_heads}, {head_dim}]")
    if dtype is _BF16:
        if k_scale is not None or v_scale is not None:
            raise ValueError("k_scale and v_scale belong to float8_e4m3fn caches")
    elif dtype is not _E4M3:
        _bad("k_pages", k, "bfloat16 or float8_e4m3fn")
    if k.get_device() != dev or ks[3] != 1:
        _bad("k_pages", k, "contiguous in its last dimension,")
    if v.shape != shape or v.dtype is not dtype or v.get_device() != dev or vs[3] != 1:
        _bad("v_pages", v, f"{dtype} {tuple(shape)}, contiguous in its last dimension,")
    return (0 if dtype is _BF16 else 1), shape, ks, vs


class AttentionWorkspace:
    """The workspace of `paged_attention` for these heads over a buffer of the caller's: contiguous uint8 on a CUDA device,
    16-byte aligned, of at least lib.paged_attn_workspace(heads, kv_heads, head_dim) bytes, all zero before its first call.
    (`attention_workspace` makes both.) A buffer elsewhere is refused by the call, as any other tensor."""

    def __init__(self, buffer, heads, kv_heads, head_dim, lib=None):
        if buffer.is_cuda:                                       # what no call checks again
            need = (load_lib() if lib is None else lib).paged_attn_workspace(heads, kv_heads, head_dim)
            if buffer.dtype is not torch.uint8 or not buffer.is_contiguous() or buffer.numel() < need or (
                    buffer.data_ptr() % 16):
                _bad("buffer", buffer, f"contiguous uint8 of at least {need} bytes, 16-byte aligned,")
        self.buffer, self.ptr, self.sizes = buffer, buffer.data_ptr(), (buffer.get_device(), heads, kv_heads, head_dim)


def attention_workspace(lib, heads, kv_heads, head_dim, device=None):
    """The zeroed workspace of `paged_attention` for these heads, for batches and lengths of any size. Calls that may
    overlap on the GPU (other streams, graphs replayed at the same time) need one each."""
    return AttentionWorkspace(torch.zeros(lib.paged_attn_workspace(heads, kv_heads, head_dim), dtype=torch.uint8,
                                          device="cuda" if device is None else device), heads, kv_heads, head_dim, lib)


def paged_attention(lib, q, k_pages, v_pages, page_table, lens, out, workspace, *, scale=None, window=0, k_scale=None,
                    v_scale=None, lse=None, stream=None):
    """out[b] = attention of q[b] (bf16 [batch, heads, head_dim]) over the first lens[b] positions of sequence b (the
    last `window` of them where window > 0). out bf16 like q; lse fp32 [batch, heads], natural logarithm, or None. A
    sequence of length 0 gets zeros and -inf. scale: 1 / sqrt(head_dim) by default."""
    if _bind is not None and _bind.paged_attention(
            lib.paged_attn_entry, lib.device_entry, q, k_pages, v_pages, page_table, lens, out, workspace.ptr,
            workspace.sizes, scale, window, k_scale, v_scale, lse, stream) == 0:
        return out
    dev, shape, qs, os = _device(q, "q"), q.shape, _strides(q), _strides(out)
    if len(shape) != 3 or q.dtype is not _BF16 or (qs[2] != 1 and shape[2] != 1):
        _bad("q", q, "bfloat16 [batch, heads, head_dim], contiguous in its last dimension,")
    if out.shape != shape or out.dtype is not _BF16 or out.get_device() != dev or os[2] != 1:
        _bad("out", out, f"bfloat16 {tuple(shape)}, contiguous in its last dimension,")
    batch, heads, hd = shape
    kv = k_pages.shape[2] if k_pages.dim() == 4 else 0
    if not kv or heads % kv:
        _bad("k_pages", k_pages, f"[num_pages, page_size, kv_heads, {hd}] with kv_heads dividing {heads}")
    cache, pool, ks, vs = _pools(k_pages, v_pages, kv, hd, k_scale, v_scale, dev)
    ts, tst = page_table.shape, _strides(page_table)
    if len(ts) != 2 or ts[0] != batch or page_table.dtype is not _I32 or page_table.get_device() != dev or (
            tst[1] != 1 and ts[1] != 1):
        _bad("page_table", page_table, f"int32 [{batch}, max_pages], contiguous in its last dimension,")
    if lens.shape != (batch,) or lens.dtype is not _I32 or lens.get_device() != dev or not lens.is_contiguous():
        _bad("lens", lens, f"contiguous int32 [{batch}]")
    lp = ls = 0
    if lse is not None:
        if lse.shape != (batch, heads) or lse.dtype is not _F32 or lse.get_device() != dev or (
                lse.stride(1) != 1 and heads != 1):
            _bad("lse", lse, f"float32 [{batch}, {heads}], contiguous in its last dimension,")
        lp, ls = lse.data_ptr(), _strides(lse)[0]
    if workspace.sizes != (dev, heads, kv, hd):
        raise ValueError(f"workspace is for (device, heads, kv_heads, head_dim) = {workspace.sizes}, the call for "
                         f"{(dev, heads, kv, hd)}")
    rc = lib.paged_attn(_pack_attn(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lens.data_ptr(),
        0 if k_scale is None else _flat("k_scale", k_scale, _F32, (kv,), dev),
        0 if v_scale is None else _flat("v_scale", v_scale, _F32, (kv,), dev), out.data_ptr(), lp, workspace.ptr,
        qs[0], qs[1], os[0], os[1], ls, tst[0], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        batch, heads, kv, hd, cache, pool[0], pool[1], ts[1], window, hd ** -0.5 if scale is None else scale),
        _raw_stream(dev) if stream is None else stream)
    if rc:
        lib._check(rc, "paia_gemv_paged_attn")
    return out


def rope_inv_freq(rot, theta, device="cuda"):
    """The plain rotary frequencies theta^(-2i / rot) as `qkv_rope_cache` takes them: fp64 [rot / 2]."""
    return float(theta) ** (-torch.arange(0, rot, 2, dtype=_F64, device=device) / rot)


def qkv_rope_cache(lib, qkv, positions, inv_freq, q_out, k_pages, v_pages, page_table, *, seq=None, q_norm=None,
                   k_norm=None, eps=1e-6, interleaved=False, k_scale=None, v_scale=None, k_out=None, kv_heads=None,
                   stream=None):
    """For each token t of qkv (bf16 [tokens, (heads + 2 kv_heads) * head_dim]): q_out[t] (bf16 [tokens, heads,
    head_dim], may be the q part of qkv) gets its q heads normed (q_norm fp32 [head_dim], None: not) and rotated at
    positions[t] (int32; -1: a padding row, left alone), and its k (normed by k_norm, rotated) and v heads go to position
    positions[t] of sequence seq[t] (int32, None: sequence t) of the paged cache. inv_freq: fp64 [rot / 2], rot <=
    head_dim (`rope_inv_freq`). k_out (bf16 [tokens, kv_heads, head_dim]) gets the rotated k heads as well; without a
    cache (k_pages, v_pages and page_table None) it is required, with kv_heads. Two rows of a call must not name the
    same sequence and position."""
    if _bind is not None and k_pages is not None and _bind.qkv_rope_cache(
            lib.qkv_rope_cache_entry, lib.device_entry, qkv, positions, inv_freq, q_out, k_pages, v_pages, page_table, seq,
            q_norm, k_norm, eps, interleaved, k_scale, v_scale, k_out, stream) == 0:
        return q_out
    dev, qs, xs = _device(qkv, "qkv"), _strides(q_out), _strides(qkv)
    if len(qs) != 3 or q_out.dtype is not _BF16 or q_out.get_device() != dev or qs[2] != 1:
        _bad("q_out", q_out, "bfloat16 [tokens, heads, head_dim], contiguous in its last dimension,")
    tokens, heads, hd = q_out.shape
    if k_pages is not None:
        kv = k_pages.shape[2] if k_pages.dim() == 4 else 0
        cache, (num_pages, page_size, _, _), ks, vs = _pools(k_pages, v_pages, kv, hd, k_scale, v_scale, dev)
        kp, vp, shape, tst = k_pages.data_ptr(), v_pages.data_ptr(), page_table.shape, _strides(page_table)
        if len(shape) != 2 or page_table.dtype is not _I32 or page_table.get_device() != dev or (
                tst[1] != 1 and shape[1] != 1) or (seq is None and shape[0] < tokens):
            _bad("page_table", page_table, "int32 [sequences, max_pages], contiguous in its last dimension,")
        seqs, max_pages = shape
        table, ts = page_table.data_ptr(), tst[0]
    else:
        if v_pages is not None or page_table is not None or k_out is None or not kv_heads:
            raise ValueError("without a cache, v_pages and page_table are None and k_out and kv_heads are given")
        kv, cache, num_pages, page_size, seqs, max_pages, table, ts, kp, vp = kv_heads, 0, 0, 1, 0, 0, 0, 0, 0, 0
        ks = vs = (0, 0, 0)
    if qkv.shape != (tokens, (heads + 2 * kv) * hd) or qkv.dtype is not _BF16 or xs[1] != 1:
        _bad("qkv", qkv, f"bfloat16 {(tokens, (heads + 2 * kv) * hd)}, contiguous in its last dimension,")
    if positions.shape != (tokens,) or positions.dtype is not _I32 or positions.get_device() != dev or (
            not positions.is_contiguous()):
        _bad("positions", positions, f"contiguous int32 [{tokens}]")
    half = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    if inv_freq.dtype is not _F64 or half < 0 or inv_freq.get_device() != dev or not inv_freq.is_contiguous():
        _bad("inv_freq", inv_freq, "contiguous float64 [rot / 2]")
    ko = kos = 0
    if k_out is not None:
        kos = _strides(k_out)
        if k_out.shape != (tokens, kv, hd) or k_out.dtype is not _BF16 or k_out.get_device() != dev or kos[2] != 1:
            _bad("k_out", k_out, f"bfloat16 {(tokens, kv, hd)}, contiguous in its last dimension,")
        ko = k_out.data_ptr()
    rc = lib.qkv_rope_cache(_pack_rope(
        qkv.data_ptr(), positions.data_ptr(), 0 if seq is None else _flat("seq", seq, _I32, (tokens,), dev),
        inv_freq.data_ptr(), 0 if q_norm is None else _flat("q_norm", q_norm, _F32, (hd,), dev),
        0 if k_norm is None else _flat("k_norm", k_norm, _F32, (hd,), dev), table,
        0 if k_scale is None else _flat("k_scale", k_scale, _F32, (kv,), dev),
        0 if v_scale is None else _flat("v_scale", v_scale, _F32, (kv,), dev), q_out.data_ptr(), ko, kp, vp,
        xs[0], qs[0], qs[1], kos[0] if ko else 0, kos[1] if ko else 0, ts, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        tokens, seqs, heads, kv, hd, 2 * half, 1 if interleaved else 0, cache, num_pages, page_size, max_pages, eps),
        _raw_stream(dev) if stream is None else stream)
    if rc:
        lib._check(rc, "paia_gemv_qkv_rope_cache")
    return q_out


def lora(lib, x, a, b, adapter, out, *, base=None, scaling=None, ranks=None, stream=None):
    """out[m] = base[m] + scaling[i] * b[i] (a[i] x[m]) for i = adapter[m] (int32; -1: out[m] = base[m]). x bf16 [M, K],
    a bf16 [adapters, rank, K], b bf16 [adapters, N, rank], out (apart from x) and base (None: zeros; may be out) bf16
    [M, N]; scaling fp32 and ranks int32 [adapters] (None: 1 and `rank`): adapter i uses its first ranks[i] ranks."""
    if _bind is not None and _bind.lora(lib.lora_entry, lib.device_entry, x, a, b, adapter, out, base, scaling, ranks,
                                        stream) == 0:
        return out
    dev, xs, sa, sb, os = _device(x, "x"), _strides(x), _strides(a), _strides(b), _strides(out)
    if len(xs) != 2 or x.dtype is not _BF16 or xs[1] != 1 or len(sa) != 3 or len(sb) != 3:
        _bad("x", x, "bfloat16 [M, K], contiguous in its last dimension (a [adapters, rank, K], b [adapters, N, rank]),")
    m, k = x.shape
    n_ad, rank, ka = a.shape
    if ka != k or a.dtype is not _BF16 or a.get_device() != dev or sa[2] != 1:
        _bad("a", a, f"bfloat16 [adapters, rank, {k}], contiguous in its last dimension,")
    n = b.shape[1]
    if b.shape != (n_ad, n, rank) or b.dtype is not _BF16 or b.get_device() != dev or sb[2] != 1:
        _bad("b", b, f"bfloat16 [{n_ad}, N, {rank}], contiguous in its last dimension,")
    if adapter.shape != (m,) or adapter.dtype is not _I32 or adapter.get_device() != dev or not adapter.is_contiguous():
        _bad("adapter", adapter, f"contiguous int32 [{m}]")
    if out.shape != (m, n) or out.dtype is not _BF16 or out.get_device() != dev or os[1] != 1:
        _bad("out", out, f"bfloat16 {(m, n)}, contiguous in its last dimension,")
    bp = bs = 0
    if base is not None:
        if base.shape != (m, n) or base.dtype is not _BF16 or base.get_device() != dev or base.stride(1) != 1:
            _bad("base", base, f"bfloat16 {(m, n)}, contiguous in its last dimension,")
        bp, bs = base.data_ptr(), _strides(base)[0]
    rc = lib.lora(_pack_lora(
        x.data_ptr(), a.data_ptr(), b.data_ptr(), adapter.data_ptr(),
        0 if ranks is None else _flat("ranks", ranks, _I32, (n_ad,), dev),
        0 if scaling is None else _flat("scaling", scaling, _F32, (n_ad,), dev), bp, out.data_ptr(),
        xs[0], bs, os[0], sa[0], sa[1], sb[0], sb[1], m, n, k, rank, n_ad),
        _raw_stream(dev) if stream is None else stream)
    if rc:
        lib._check(rc, "paia_gemv_lora")
    return out


class Routing:
    """Where `route` writes for up to `tokens` tokens: weights fp32 [tokens, top_k], experts and places int32 [tokens, top_k],
    rows int32 [tokens * top_k], offsets int32 [experts + 1], on one CUDA device, and its workspace. (`routing` makes one.)
    first(n) is the same for the first n tokens, over the same memory."""

    def __init__(self, lib, weights, experts, places, rows, offsets, workspace):
        self.lib, self.weights, self.experts, self.places, self.rows = lib, weights, experts, places, rows
        self.offsets, self.workspace = offsets, workspace
        dev, (tokens, top_k), n = weights.get_device(), weights.shape, offsets.shape[0] - 1
        need = lib.route_workspace(n) if weights.is_cuda else 0
        for name, t, dtype, shape in (("weights", weights, _F32, (tokens, top_k)), ("experts", experts, _I32, (tokens, top_k)),
                                      ("places", places, _I32, (tokens, top_k)), ("rows", rows, _I32, (tokens * top_k,)),
                                      ("offsets", offsets, _I32, (n + 1,)), ("workspace", workspace, _U8, workspace.shape)):
            if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
                _bad(name, t, f"contiguous {dtype} {shape}")
        if workspace.numel() < need or workspace.data_ptr() % 16:
            _bad("workspace", workspace, f"contiguous uint8 of at least {need} bytes, 16-byte aligned,")
        self.ptrs = tuple(t.data_ptr() for t in (weights, experts, places, rows, offsets, workspace))
        self.sizes = (dev, tokens, n, top_k)

    def first(self, n):
        k = self.sizes[3]
        return Routing(self.lib, self.weights[:n], self.experts[:n], self.places[:n], self.rows[:n * k], self.offsets,
                       self.workspace)


def routing(lib, tokens, experts, top_k, device=None):
    """A `Routing` for up to `tokens` tokens. Calls that may overlap on the GPU need one each."""
    dev = "cuda" if device is None else device
    i32 = lambda *shape: torch.zeros(*shape, dtype=_I32, device=dev)   # noqa: E731
    return Routing(lib, torch.zeros(tokens, top_k, dtype=_F32, device=dev), i32(tokens, top_k), i32(tokens, top_k),
                   i32(tokens * top_k), i32(experts + 1), torch.zeros(lib.route_workspace(experts), dtype=_U8, device=dev))


_SCORING = {"softmax": 0, "sigmoid": 1}


def route(lib, logits, routing, *, scoring="softmax", bias=None, renormalise=True, scale=1.0, positions=None, stream=None):
    """Each token's top_k experts by its logits (bf16 or fp32 [tokens, experts]), in falling order (ties to the lowest index),
    their weights (times `scale`), and the tokens grouped by expert, into `routing`. scoring "softmax": weights e^l over the
    sum of the chosen (renormalise) or of all; "sigmoid": ordered by sigmoid(l) + bias (fp32 [experts] or None), weights
    sigmoid(l), over the sum of the chosen where renormalise. positions (int32 [tokens], None: all live): rows below 0 are
    padding, with experts and places -1 and no place among the rows."""
    if _bind is not None and _bind.route(lib.route_entry, lib.device_entry, logits, routing.ptrs, routing.sizes, scoring, bias,
                                         renormalise, scale, positions, stream) == 0:
        return routing
    dev, ls = _device(logits, "logits"), _strides(logits)
    sizes = routing.sizes
    if logits.dtype not in (_BF16, _F32) or logits.shape != sizes[1:3] or (ls[1] != 1 and sizes[2] != 1):
        _bad("logits", logits, f"bfloat16 or float32 {sizes[1:3]}, contiguous in its last dimension,")
    if sizes[0] != dev:
        raise ValueError(f"routing is on device {sizes[0]}, the call on {dev}")
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {tuple(_SCORING)}, got {scoring!r}")
    if bias is not None and scoring != "sigmoid":
        raise ValueError("bias belongs to sigmoid scoring")
    weights, experts, places, rows, offsets, workspace = routing.ptrs
    rc = lib.route(_pack_route(
        logits.data_ptr(), _flat("bias", bias, _F32, (sizes[2],), dev), _flat("positions", positions, _I32, (sizes[1],), dev),
        weights, experts, places, rows, offsets, workspace, ls[0], sizes[1], sizes[2], sizes[3],
        0 if logits.dtype is _BF16 else 1, _SCORING[scoring], 1 if renormalise else 0, scale),
        _raw_stream(dev) if stream is None else stream)
    if rc:
        lib._check(rc, "paia_gemv_route")
    return routing


class ExpertWorkspace:
    """The workspace of `expert_matmul` over a buffer of the caller's: contiguous uint8 on a CUDA device, 16-byte aligned, of
    at least lib.expert_workspace() bytes, all zero before its first call. (`expert_workspace` makes both.)"""

    def __init__(self, buffer, lib=None):
        if buffer.is_cuda:
            need = (load_lib() if lib is None else lib).expert_workspace()
            if buffer.dtype is not _U8 or not buffer.is_contiguous() or buffer.numel() < need or buffer.data_ptr() % 16:
                _bad("buffer", buffer, f"contiguous uint8 of at least {need} bytes, 16-byte aligned,")
        self.buffer, self.ptr, self.device = buffer, buffer.data_ptr(), buffer.get_device()


def expert_workspace(lib, device=None):
    """The zeroed workspace of `expert_matmul`, for calls of any sizes. Calls that may overlap on the GPU need one each."""
    return ExpertWorkspace(torch.zeros(lib.expert_workspace(), dtype=_U8, device="cuda" if device is None else device), lib)


def expert_matmul(lib, w, x, offsets, out, workspace, *, scales=None, rows=None, silu=False, stream=None):
    """out[i] = w[e] x[rows[i]] for i in offsets[e] .. offsets[e + 1] - 1 of every expert e (int32 [experts + 1]; `route`
    makes offsets and rows). w [experts, N, K] bf16, or e4m3 (float8_e4m3fn or its bytes as uint8) with scales fp32
    [experts, N]; x bf16 [rows, K]; rows int32 [M] (None: x[i]); out bf16 [M, N] (apart from x). silu: w[e] holds [gate; up]
    and out [M, N / 2] gets silu(gate x) * (up x). Rows of out that belong to no expert stay as they were."""
    if _bind is not None and _bind.expert_matmul(lib.expert_matmul_entry, lib.device_entry, w, x, offsets, out, workspace.ptr,
                                                 workspace.device, scales, rows, silu, stream) == 0:
        return out
    dev, sw, xs, os = _device(x, "x"), _strides(w), _strides(x), _strides(out)
    if len(xs) != 2 or x.dtype is not _BF16 or xs[1] != 1:
        _bad("x", x, "bfloat16 [rows, K], contiguous in its last dimension,")
    kind = 0 if w.dtype is _BF16 else 1
    if len(sw) != 3 or w.dtype not in (_BF16, _E4M3, _U8) or w.get_device() != dev or sw[2] != 1 or w.shape[2] != x.shape[1]:
        _bad("w", w, f"bfloat16, float8_e4m3fn or uint8 [experts, N, {x.shape[1]}], contiguous in its last dimension,")
    e, n, k = w.shape
    ss = (0, 1)
    if kind == 1:
        if scales is None or scales.shape != (e, n) or scales.dtype is not _F32 or scales.get_device() != dev:
            _bad("scales", scales, f"float32 {(e, n)}")
        ss = _strides(scales)
        if ss[1] != 1 and n != 1:
            _bad("scales", scales, f"float32 {(e, n)}, contiguous in its last dimension,")
    elif scales is not None:
        raise ValueError("scales belong to e4m3 weights")
    if silu and n % 2:
        raise ValueError(f"with silu w holds gate and up: N must be even, got {n}")
    cols = n // 2 if silu else n
    if len(os) != 2 or out.shape[1] != cols or out.dtype is not _BF16 or out.get_device() != dev or (os[1] != 1 and cols != 1):
        _bad("out", out, f"bfloat16 [M, {cols}], contiguous in its last dimension,")
    m = out.shape[0]
    if offsets.shape != (e + 1,) or offsets.dtype is not _I32 or offsets.get_device() != dev or not offsets.is_contiguous():
        _bad("offsets", offsets, f"contiguous int32 [{e + 1}]")
    if rows is None and x.shape[0] < m:
        _bad("x", x, f"bfloat16 [at least {m}, {k}] where rows is None")
    if workspace.device != dev:
        raise ValueError(f"workspace is on device {workspace.device}, the call on {dev}")
    rc = lib.expert_matmul(_pack_experts(
        w.data_ptr(), 0 if scales is None else scales.data_ptr(), x.data_ptr(), _flat("rows", rows, _I32, (m,), dev),
        offsets.data_ptr(), out.data_ptr(), workspace.ptr, sw[0], sw[1] if n > 1 else k, xs[0], os[0], ss[0], e, m, n, k,
        x.shape[0], kind, 1 if silu else 0, 0), _raw_stream(dev) if stream is None else stream)
    if rc:
        lib._check(rc, "paia_gemv_expert_matmul")
    return out


def block_norm(lib, h, x=None, h_out=None, *, out=None, places=None, weights=None, post=None, gate=None, scale=1.0, pre=None,
               eps=1e-5, stream=None):
    """h_out[t] = h[t] + scale * gate * norm(y[t]), y[t] = x[t], or sum_j weights[t, j] x[places[t, j]] (int32 and fp32
    [tokens, top_k]; a place of -1 adds nothing), norm(y) = y / sqrt(mean y^2 + eps) * post (post fp32 [hidden]; None: y as
    it is); out[t] = h_out[t] / sqrt(mean h_out[t]^2 + eps) * pre where out and pre (fp32 [hidden]) are given. h, x, h_out,
    out bf16 [.., hidden]; h_out may be h. gate bf16 [hidden], [tokens, 1] or [tokens, hidden]. Without x (and h_out): the
    norm of h alone."""
    if _bind is not None and _bind.block_norm(lib.block_norm_entry, lib.device_entry, h, x, h_out, out, places, weights, post,
                                              gate, scale, pre, eps, stream) == 0:
        return out if h_out is None else h_out
    dev, hs = _device(h, "h"), _strides(h)
    if len(hs) != 2 or h.dtype is not _BF16 or hs[1] != 1:
        _bad("h", h, "bfloat16 [tokens, hidden], contiguous in its last dimension,")
    t, hid = h.shape

    def like(name, v, n):
        if v is None:
            return 0, 0
        s = _strides(v)
        if len(s) != 2 or (v.shape[0] < t if n is None else v.shape[0] != n) or v.shape[1] != hid or v.dtype is not _BF16 or (
                v.get_device() != dev or s[1] != 1):
            _bad(name, v, f"bfloat16 [{'rows' if n is None else n}, {hid}], contiguous in its last dimension,")
        return v.data_ptr(), s[0]

    top_k, ps, wts = 0, 0, 0
    if places is not None:
        if len(places.shape) != 2 or places.shape[0] != t or places.shape[1] < 1 or places.dtype is not _I32 or (
                places.get_device() != dev or places.stride(1) != 1 and places.shape[1] != 1):
            _bad("places", places, f"int32 [{t}, top_k >= 1], contiguous in its last dimension,")
        top_k = places.shape[1]
        if weights is None or weights.shape != places.shape or weights.dtype is not _F32 or weights.get_device() != dev or (
                weights.stride(1) != 1 and top_k != 1):
            _bad("weights", weights, f"float32 {(t, top_k)}, contiguous in its last dimension,")
        ps, wts = _strides(places)[0], _strides(weights)[0]
    elif weights is not None:
        raise ValueError("weights belong to places")
    if x is not None and x.dim() == 2 and places is not None:
        if x.shape[1] != hid or x.dtype is not _BF16 or x.get_device() != dev or _strides(x)[1] != 1:
            _bad("x", x, f"bfloat16 [rows, {hid}], contiguous in its last dimension,")
        xp, xs = x.data_ptr(), _strides(x)[0]
    else:
        xp, xs = like("x", x, None)
    op, os = like("h_out", h_out, t)
    np, ns = like("out", out, t)
    gp = gs = gc = 0
    if gate is not None:
        shape, s = gate.shape, _strides(gate)
        if gate.dtype is not _BF16 or gate.get_device() != dev or shape not in ((hid,), (t, 1), (t, hid)) or (
                s[-1] != 1 and shape[-1] != 1):
            _bad("gate", gate, f"bfloat16 {(hid,)}, {(t, 1)} or {(t, hid)}, contiguous in its last dimension,")
        gp, gs, gc = gate.data_ptr(), s[0] if len(s) == 2 else 0, 1 if shape[-1] == hid else 0
    if (x is None) != (h_out is None):
        raise ValueError("x and h_out go together")
    rc = lib.block_norm(_pack_norm(
        xp, h.data_ptr(), op, np, 0 if places is None else places.data_ptr(), 0 if weights is None else weights.data_ptr(),
        _flat("post", post, _F32, (hid,), dev), _flat("pre", pre, _F32, (hid,), dev), gp, xs, hs[0], os, ns, ps, wts, gs, t, hid,
        top_k, 0 if x is None else x.shape[0], gc, eps, scale, 0), _raw_stream(dev) if stream is None else stream)
    if rc:
        lib._check(rc, "paia_gemv_block_norm")
    return out if h_out is None else h_out
