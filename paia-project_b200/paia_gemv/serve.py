"""Serving operators on torch tensors: what a batched decode step does between its GEMVs (include/paia_gemv.h has the
definitions). Each call checks its tensors, packs the C struct and launches on torch's current stream (or `stream`);
outputs are written in place, nothing is allocated and nothing synchronises, so every call is CUDA-graph capturable.

    qkv_rope_cache   per-head norm, rotary positions and cache write of a fused QKV projection's rows
    paged_attention  attention of one new token per sequence over the paged cache
    lora             the low-rank adapters of many requests, added to a shared projection

Caches are a pair of tensors [num_pages, page_size, kv_heads, head_dim] (bf16, or float8_e4m3fn with a fp32 scale per
kv head), in any layout whose head_dim is contiguous: a [num_pages, kv_heads, page_size, head_dim] pool is passed as
`pool.transpose(1, 2)`. Page tables are int32 [sequences, max_pages]. Tensors live on the current CUDA device.
"""
import struct

import torch

# the C structs, field by field (native alignment): include/paia_gemv.h
ATTN = struct.Struct("10P 12q 9i f")
ROPE_CACHE = struct.Struct("13P 12q 11i f")
LORA = struct.Struct("8P 7q 5i 4x")

_BF16, _F32, _F64, _I32, _E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.float8_e4m3fn


def _bad(name, t, what):
    raise ValueError(f"{name} must be {what}, got " + (f"{t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}"
                                                       if isinstance(t, torch.Tensor) else repr(t)))


def _rows(name, t, dtype, shape, dev):
    """t: `shape`, contiguous innermost dimension, any other strides."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != dev or (t.stride()[-1] != 1 and shape[-1] != 1):
        _bad(name, t, f"{dtype} {tuple(shape)} on the current CUDA device, contiguous in its last dimension")
    return t.data_ptr()


def _flat(name, t, dtype, n, dev):
    """Contiguous [n], or None."""
    if t is None:
        return 0
    if t.shape != (n,) or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        _bad(name, t, f"contiguous {dtype} [{n}] on the current CUDA device")
    return t.data_ptr()


def _device(t, name):
    dev = t.get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}: the operators run on the current CUDA device")
    return dev


def _pools(k, v, kv_heads, head_dim, k_scale, v_scale, dev):
    """(cache code, pool shape) of a cache's two pools."""
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or shape[2] != kv_heads or shape[3] != head_dim:
        _bad("k_pages", k, f"[num_pages, page_size, {kv_heads}, {head_dim}]")
    if dtype is not _BF16 and dtype is not _E4M3:
        _bad("k_pages", k, "bfloat16 or float8_e4m3fn")
    if dtype is _BF16 and (k_scale is not None or v_scale is not None):
        raise ValueError("k_scale and v_scale belong to float8_e4m3fn caches")
    if k.get_device() != dev or k.stride()[3] != 1:
        _bad("k_pages", k, "on the current CUDA device, contiguous in its last dimension")
    if v.shape != shape or v.dtype is not dtype or v.get_device() != dev or v.stride()[3] != 1:
        _bad("v_pages", v, f"{dtype} {tuple(shape)} on the current CUDA device, contiguous in its last dimension")
    return (0 if dtype is _BF16 else 1), shape


class AttentionWorkspace:
    """The workspace of `paged_attention` for these heads (`attention_workspace` makes it)."""

    def __init__(self, buffer, heads, kv_heads, head_dim):
        self.buffer, self.ptr, self.sizes = buffer, buffer.data_ptr(), (buffer.get_device(), heads, kv_heads, head_dim)


def attention_workspace(lib, heads, kv_heads, head_dim, device=None):
    """The zeroed workspace of `paged_attention` for these heads, for batches and lengths of any size. Calls that may
    overlap on the GPU (other streams, graphs replayed at the same time) need one each."""
    return AttentionWorkspace(torch.zeros(lib.paged_attn_workspace(heads, kv_heads, head_dim), dtype=torch.uint8,
                                          device="cuda" if device is None else device), heads, kv_heads, head_dim)


def paged_attention(lib, q, k_pages, v_pages, page_table, lens, out, workspace, *, scale=None, window=0, k_scale=None,
                    v_scale=None, lse=None, stream=None):
    """out[b] = attention of q[b] (bf16 [batch, heads, head_dim]) over the first lens[b] positions of sequence b (the
    last `window` of them where window > 0). out bf16 like q; lse fp32 [batch, heads], natural logarithm, or None. A
    sequence of length 0 gets zeros and -inf. scale: 1 / sqrt(head_dim) by default."""
    dev, shape, pool = _device(q, "q"), q.shape, k_pages.shape
    if len(shape) != 3:
        _bad("q", q, "[batch, heads, head_dim]")
    batch, heads, hd = shape
    kv = pool[2] if len(pool) == 4 else 0
    if not kv or heads % kv:
        _bad("k_pages", k_pages, f"[num_pages, page_size, kv_heads, {hd}] with kv_heads dividing {heads}")
    cache, pool = _pools(k_pages, v_pages, kv, hd, k_scale, v_scale, dev)
    ts = page_table.shape
    if len(ts) != 2 or ts[0] != batch:
        _bad("page_table", page_table, f"[{batch}, max_pages]")
    table = _rows("page_table", page_table, _I32, ts, dev)
    if workspace.sizes != (dev, heads, kv, hd):
        raise ValueError(f"workspace is for (device, heads, kv_heads, head_dim) = {workspace.sizes}, the call for "
                         f"{(dev, heads, kv, hd)}")
    ks, vs = k_pages.stride(), v_pages.stride()
    qs, os = q.stride(), out.stride()
    lib.paged_attn(ATTN.pack(
        _rows("q", q, _BF16, shape, dev), k_pages.data_ptr(), v_pages.data_ptr(), table,
        _flat("lens", lens, _I32, batch, dev), _flat("k_scale", k_scale, _F32, kv, dev),
        _flat("v_scale", v_scale, _F32, kv, dev), _rows("out", out, _BF16, shape, dev),
        0 if lse is None else _rows("lse", lse, _F32, (batch, heads), dev), workspace.ptr,
        qs[0], qs[1], os[0], os[1], 0 if lse is None else lse.stride(0), page_table.stride(0),
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        batch, heads, kv, hd, cache, pool[0], pool[1], ts[1], window,
        hd ** -0.5 if scale is None else scale), torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream)
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
    dev = _device(qkv, "qkv")
    if q_out.dim() != 3 or qkv.dim() != 2:
        _bad("qkv and q_out", q_out, "[tokens, (heads + 2 kv_heads) * head_dim] and [tokens, heads, head_dim]")
    tokens, heads, hd = q_out.shape
    if k_pages is not None:
        kv = k_pages.shape[2] if k_pages.dim() == 4 else 0
        cache, (num_pages, page_size, _, _) = _pools(k_pages, v_pages, kv, hd, k_scale, v_scale, dev)
        ks, vs, kp, vp = k_pages.stride(), v_pages.stride(), k_pages.data_ptr(), v_pages.data_ptr()
        if page_table.dim() != 2 or (seq is None and page_table.shape[0] < tokens):
            _bad("page_table", page_table, "[sequences, max_pages]")
        seqs, max_pages = page_table.shape
        table, ts = _rows("page_table", page_table, _I32, page_table.shape, dev), page_table.stride(0)
    else:
        if v_pages is not None or page_table is not None or k_out is None or not kv_heads:
            raise ValueError("without a cache, v_pages and page_table are None and k_out and kv_heads are given")
        kv, cache, num_pages, page_size, seqs, max_pages, table, ts, kp, vp = kv_heads, 0, 0, 1, 0, 0, 0, 0, 0, 0
        ks = vs = (0, 0, 0)
    qs = q_out.stride()
    kos = (0, 0) if k_out is None else k_out.stride()
    half = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    lib.qkv_rope_cache(ROPE_CACHE.pack(
        _rows("qkv", qkv, _BF16, (tokens, (heads + 2 * kv) * hd), dev),
        _flat("positions", positions, _I32, tokens, dev), _flat("seq", seq, _I32, tokens, dev),
        _flat("inv_freq", inv_freq, _F64, half, dev), _flat("q_norm", q_norm, _F32, hd, dev),
        _flat("k_norm", k_norm, _F32, hd, dev), table, _flat("k_scale", k_scale, _F32, kv, dev),
        _flat("v_scale", v_scale, _F32, kv, dev), _rows("q_out", q_out, _BF16, (tokens, heads, hd), dev),
        0 if k_out is None else _rows("k_out", k_out, _BF16, (tokens, kv, hd), dev), kp, vp,
        qkv.stride(0), qs[0], qs[1], kos[0], kos[1], ts, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        tokens, seqs, heads, kv, hd, 2 * half, 1 if interleaved else 0, cache, num_pages, page_size, max_pages, eps),
        torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream)
    return q_out


def lora(lib, x, a, b, adapter, out, *, base=None, scaling=None, ranks=None, stream=None):
    """out[m] = base[m] + scaling[i] * b[i] (a[i] x[m]) for i = adapter[m] (int32; -1: out[m] = base[m]). x bf16 [M, K],
    a bf16 [adapters, rank, K], b bf16 [adapters, N, rank], out and base (None: zeros; may be out) bf16 [M, N]; scaling
    fp32 and ranks int32 [adapters] (None: 1 and `rank`): adapter i uses its first ranks[i] ranks."""
    dev = _device(x, "x")
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        _bad("x, a and b", x, "[M, K], [adapters, rank, K] and [adapters, N, rank]")
    m, k = x.shape
    n_ad, rank, n = a.shape[0], a.shape[1], b.shape[1]
    sa, sb = a.stride(), b.stride()
    lib.lora(LORA.pack(
        _rows("x", x, _BF16, (m, k), dev), _rows("a", a, _BF16, (n_ad, rank, k), dev),
        _rows("b", b, _BF16, (n_ad, n, rank), dev), _flat("adapter", adapter, _I32, m, dev),
        _flat("ranks", ranks, _I32, n_ad, dev), _flat("scaling", scaling, _F32, n_ad, dev),
        0 if base is None else _rows("base", base, _BF16, (m, n), dev), _rows("out", out, _BF16, (m, n), dev),
        x.stride(0), 0 if base is None else base.stride(0), out.stride(0), sa[0], sa[1], sb[0], sb[1],
        m, n, k, rank, n_ad), torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream)
    return out
