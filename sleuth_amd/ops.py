"""Torch-tensor front ends of the HIP kernels (C ABI in include/forge_attn.h).

These functions only check shapes on the host, pick pointers/strides and launch on
torch's current stream; calls whose arguments need no conversion are checked and launched by the
native host module (csrc/host.cpp), which returns None for the others. They never compute anything themselves: if the library is not
built they raise (sleuth_amd._lib.ForgeError).

Layouts (reference names): q [B,H,T,D] (any strides, last dim contiguous: the transposed
q_proj view, attention.py:106), k/v [B,K,T,D], caches [B,K,max_len,D] (kv_cache.py:31),
outputs [B,T,H,D] (attention.py:155).
"""

from __future__ import annotations

import contextlib

import torch

from . import _lib
from ._lib import BF16, F16, F32, FIXED_CUT, NORM_QK, NORM_V, ROPE, WS_ZEROED, check, host, lib

_DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype} (float32, bfloat16, float16)") from None


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _need_device(*ts: torch.Tensor | None) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError("forge kernels need tensors on the GPU")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must be on the same GPU")
    assert dev is not None
    return dev


def _last_dim_contiguous(t: torch.Tensor, name: str) -> None:
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")


def _weight(w: torch.Tensor | None, D: int) -> torch.Tensor | None:
    if w is None:
        return None
    if w.numel() != D:
        raise ValueError(f"norm gain has {w.numel()} values for head dim {D}")
    w = w.detach()
    if w.dtype == torch.float32 and w.is_contiguous():
        return w
    return w.to(torch.float32).contiguous()


def _rope_tables(cos, sin, B: int, T: int, D: int):
    """cos/sin [T, D] (shared positions) or [B, T, D] (per row) fp32 -> (cos, sin, s_b, s_t)."""
    if cos is None and sin is None:
        return None, None, 0, 0
    if cos is None or sin is None:
        raise ValueError("cos and sin must both be given")
    if cos.shape != sin.shape or cos.shape[-1] != D or cos.shape[-2] != T or cos.dim() not in (2, 3):
        raise ValueError(f"cos/sin must be [T, D] or [B, T, D] with T={T}, D={D}; got {tuple(cos.shape)}")
    if cos.dim() == 3 and cos.shape[0] not in (1, B):
        raise ValueError("per-row cos/sin need batch size B")
    cos = cos.to(torch.float32)
    sin = sin.to(torch.float32)
    if cos.stride(-1) != 1:
        cos = cos.contiguous()
    if sin.stride() != cos.stride():
        sin = sin.contiguous()
        cos = cos.contiguous()
    s_b = cos.stride(0) if cos.dim() == 3 and cos.shape[0] == B and B > 1 else 0
    return cos, sin, s_b, cos.stride(-2)


def _positions(pos, pos_dev, row_pos, B: int, device):
    """(row_pos int32 [B] | None, pos_dev int64 [1] | None, pos0 int)."""
    if row_pos is not None:
        if row_pos.dtype != torch.int32 or row_pos.numel() != B or row_pos.device != device:
            raise ValueError("row_pos must be an int32 [B] tensor on the GPU")
        return row_pos.contiguous(), None, 0
    if pos_dev is not None:
        if pos_dev.dtype != torch.int64 or pos_dev.device != device:
            raise ValueError("pos_dev must be an int64 tensor on the GPU")
        return None, pos_dev, 0
    return None, None, int(pos or 0)


def head_norm_rope(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6,
                   cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                   norm: bool = True) -> torch.Tensor:
    """fused_ops.head_norm_rope (fused_ops.py:101-121): x [B,H,T,D] -> per-head RMSNorm
    (gain `weight`, if norm) then NEOX RoPE (if cos/sin), one rounding; same layout as x."""
    B, H, T, D = x.shape
    dev = _need_device(x, cos, sin)
    if x.stride(-1) != 1:
        x = x.contiguous()
    y = torch.empty_like(x)
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    w = _weight(weight, D)
    st = lib().forge_head_norm_rope(dtype_code(x), _ptr(x), _ptr(y), B, H, T, D,
                                    x.stride(0), x.stride(1), x.stride(2),
                                    y.stride(0), y.stride(1), y.stride(2),
                                    _ptr(w), float(eps), int(bool(norm)),
                                    _ptr(c), _ptr(s), s_b, s_t, _stream(dev))
    check(st, "forge_head_norm_rope")
    return y


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
              pos: int | None = None, pos_dev: torch.Tensor | None = None,
              row_pos: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
              eps: float = 1e-6, norm_k: bool = False, norm_v: bool = False,
              cos: torch.Tensor | None = None, sin: torch.Tensor | None = None) -> None:
    """Normalise/rotate the new k (and v_norm v) and write them into the cache at
    base_b + t (KVCache.update, kv_cache.py:52-60; StaticKVCache.update 107-114)."""
    if pos_dev is None and row_pos is None:
        st = host().kv_append(k, v, k_cache, v_cache, int(pos or 0), k_weight, float(eps), bool(norm_k), bool(norm_v),
                              cos, sin)
        if st is not None:
            return check(st, "forge_kv_append")
    B, K, T, D = k.shape
    if v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    if k_cache.shape != v_cache.shape or k_cache.dim() != 4 or k_cache.shape[0] != B or \
            k_cache.shape[1] != K or k_cache.shape[3] != D:
        raise ValueError(f"cache {tuple(k_cache.shape)} does not fit new k {tuple(k.shape)}")
    if k_cache.stride() != v_cache.stride():
        raise ValueError("k and v caches must have the same strides")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        k, v = k.to(k_cache.dtype), v.to(k_cache.dtype)
    dev = _need_device(k, v, k_cache, v_cache, cos, sin)
    for t, n in ((k, "k"), (v, "v"), (k_cache, "k_cache")):
        _last_dim_contiguous(t, n)
    rp, pd, p0 = _positions(pos, pos_dev, row_pos, B, dev)
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    flags = (NORM_QK if norm_k else 0) | (ROPE if c is not None else 0) | (NORM_V if norm_v else 0)
    w = _weight(k_weight, D) if norm_k else None
    st = lib().forge_kv_append(dtype_code(k_cache), B, T, K, D,
                               _ptr(k), k.stride(0), k.stride(1), k.stride(2),
                               _ptr(v), v.stride(0), v.stride(1), v.stride(2),
                               _ptr(k_cache), _ptr(v_cache), k_cache.stride(0), k_cache.stride(1),
                               k_cache.stride(2), k_cache.shape[2], _ptr(rp), _ptr(pd), p0,
                               _ptr(w), float(eps), flags, _ptr(c), _ptr(s), s_b, s_t, _stream(dev))
    check(st, "forge_kv_append")


DECODE_CHUNK_MAX_T = 16  # the longest verify step the chunk span allows for (as the C default)


def decode_chunk(dtype: torch.dtype, B: int, T: int, H: int, K: int, D: int, max_kv_len: int,
                 window: int = 0, uniform: bool = False) -> int:
    """Default split-K chunk. T does not enter (decode and verify of a model share chunk
    boundaries, so verify rows equal single-token decodes bit for bit); with a sliding window
    it is sized for the keys a row can see, window + 16, not the cache length. `uniform`:
    every row of the calls starts at one position (`pos`, or `pos_dev` on the device), so
    rows have one length and the chunk only spreads the work over the CUs
    (forge_attn_decode_chunk_uniform)."""
    span = int(max_kv_len)
    if window > 0 and window + DECODE_CHUNK_MAX_T < span:
        span = window + DECODE_CHUNK_MAX_T
    fn = lib().forge_attn_decode_chunk_uniform if uniform else lib().forge_attn_decode_chunk
    return fn(_DTYPES[dtype], B, T, H, K, D, span)


def decode_workspace_bytes(dtype: torch.dtype, B: int, T: int, H: int, K: int, D: int,
                           max_kv_len: int, chunk: int = 0) -> int:
    return lib().forge_attn_decode_workspace_bytes(_DTYPES[dtype], B, T, H, K, D, int(max_kv_len), int(chunk))


def _decode_args(q, k_cache, v_cache, scale, pos, pos_dev, row_pos, max_kv_len, window, q_weight,
                 eps, norm_q, cos, sin, chunk, out, workspace):
    """Host checks of a decode call; returns (C arguments up to `out`'s strides, out,
    device, max_kv_len, chunk)."""
    B, H, T, D = q.shape
    Bc, K, max_len, Dc = k_cache.shape
    if Bc != B or Dc != D or v_cache.shape != k_cache.shape or H % K:
        raise ValueError(f"q {tuple(q.shape)} does not fit cache {tuple(k_cache.shape)}")
    if k_cache.stride() != v_cache.stride():
        raise ValueError("k and v caches must have the same strides")
    if q.dtype != k_cache.dtype:
        raise ValueError(f"q is {q.dtype} but the cache is {k_cache.dtype}")
    dev = _need_device(q, k_cache, v_cache, cos, sin, out, workspace)
    _last_dim_contiguous(q, "q")
    _last_dim_contiguous(k_cache, "k_cache")
    rp, pd, p0 = _positions(pos, pos_dev, row_pos, B, dev)
    if max_kv_len is None:
        max_kv_len = p0 + T if (rp is None and pd is None) else max_len
    max_kv_len = max(1, min(int(max_kv_len), max_len))
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    flags = (NORM_QK if norm_q else 0) | (ROPE if c is not None else 0)
    w = _weight(q_weight, D) if norm_q else None
    if out is None:
        out = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    elif out.shape != (B, T, H, D) or out.dtype != q.dtype:
        raise ValueError(f"out must be [B,T,H,D] = {(B, T, H, D)} {q.dtype}")
    if chunk <= 0:  # from the cache's capacity, not this call's length: stable across steps
        chunk = decode_chunk(q.dtype, B, T, H, K, D, max_len, window, uniform=rp is None)
    args = (dtype_code(q), B, T, H, K, D, _ptr(q), q.stride(0), q.stride(1), q.stride(2),
            _ptr(w), float(eps), flags, _ptr(c), _ptr(s), s_b, s_t,
            _ptr(k_cache), _ptr(v_cache), k_cache.stride(0), k_cache.stride(1),
            k_cache.stride(2), max_len, _ptr(rp), _ptr(pd), p0, max_kv_len,
            int(window), float(scale), int(chunk),
            _ptr(out), out.stride(0), out.stride(1), out.stride(2))
    return args, out, dev, max_kv_len, chunk


def attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, scale: float,
                pos: int | None = None, pos_dev: torch.Tensor | None = None,
                row_pos: torch.Tensor | None = None, max_kv_len: int | None = None,
                window: int = 0, q_weight: torch.Tensor | None = None, eps: float = 1e-6,
                norm_q: bool = False, cos: torch.Tensor | None = None,
                sin: torch.Tensor | None = None, chunk: int = 0, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Split-K attention of the T new queries q [B,H,T,D] against the cache, whose rows
    hold base_b + T valid keys (the new ones included). Returns [B,T,H,D]."""
    args, out, dev, max_kv_len, chunk = _decode_args(q, k_cache, v_cache, scale, pos, pos_dev, row_pos,
                                                     max_kv_len, window, q_weight, eps, norm_q, cos, sin,
                                                     chunk, out, workspace)
    B, H, T, D = q.shape
    need = lib().forge_attn_decode_workspace_bytes(args[0], B, T, H, k_cache.shape[1], D, max_kv_len, chunk)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    st = lib().forge_attn_decode(*args, _ptr(workspace), ws_bytes, _stream(dev))
    check(st, "forge_attn_decode")
    return out


_STREAM_WS: dict = {}
_PAGED_WS: dict = {}      # the same for attn_paged and attn_sinks, whose workspaces begin with other counters
_STREAM_WS_MAX = 16   # streams whose workspace is kept (the oldest is dropped beyond that)


def _take_stream_workspace(dev: torch.device, need: int, table: dict = _STREAM_WS) -> tuple[tuple, torch.Tensor]:
    """A split-K workspace per (device, stream), cleared when it is made: every call leaves
    its work ticket zero, so calls ordered on that stream may skip the ticket reset. Grown
    (a new cleared buffer) when a call needs more. It is out of the table until the call is
    launched (_put_back_stream_workspace): another thread on the stream makes one of its own
    rather than launch between this call's kernels. Dropping a buffer is safe while its calls
    are in flight: torch's allocator reuses the memory only in that stream's order."""
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = table.pop(key, None)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=dev)
    return key, ws


def _put_back_stream_workspace(key: tuple, ws: torch.Tensor, table: dict = _STREAM_WS) -> None:
    table[key] = ws   # most recently used last
    for old in list(table)[:-_STREAM_WS_MAX]:
        table.pop(old, None)


def attn_decode_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, *, scale: float, pos: int | None = None,
                       pos_dev: torch.Tensor | None = None, row_pos: torch.Tensor | None = None,
                       max_kv_len: int | None = None, window: int = 0,
                       q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                       eps: float = 1e-6, norm_q: bool = False, norm_k: bool = False,
                       norm_v: bool = False, cos: torch.Tensor | None = None,
                       sin: torch.Tensor | None = None, chunk: int = 0, out: torch.Tensor | None = None,
                       workspace: torch.Tensor | None = None, workspace_zeroed: bool = False) -> torch.Tensor:
    """kv_append(k, v, ...) then attn_decode(q, ...), as one forge_attn_decode_append call:
    the new keys (norm_k with k_weight, RoPE) and values (norm_v) go into the cache at
    base_b + t and the T queries attend over it, the new keys included. Returns [B,T,H,D].
    Without a workspace (and outside graph capture) the call uses this module's zeroed
    workspace for the current stream (FORGE_WS_ZEROED: no ticket-reset kernel);
    workspace_zeroed=True makes the same promise for a workspace the caller cleared once."""
    if out is None and workspace is None:
        r = host().decode_append(_STREAM_WS, q, k, v, k_cache, v_cache, float(scale), pos, pos_dev, row_pos, max_kv_len,
                                 window, q_weight, k_weight, float(eps), bool(norm_q), bool(norm_k), bool(norm_v), cos,
                                 sin, chunk)
        if r is not None:
            return r if r.__class__ is not int else check(r, "forge_attn_decode_append")
    B, K, T, D = k.shape
    if v.shape != k.shape or q.shape[0] != B or q.shape[2] != T or q.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    if k_cache.shape[1] != K:
        raise ValueError(f"cache {tuple(k_cache.shape)} does not fit new k {tuple(k.shape)}")
    if k.dtype != k_cache.dtype:
        k = k.to(k_cache.dtype)
    if v.dtype != k_cache.dtype:
        v = v.to(k_cache.dtype)
    _need_device(k, v)
    _last_dim_contiguous(k, "k")
    _last_dim_contiguous(v, "v")
    args, out, dev, max_kv_len, chunk = _decode_args(q, k_cache, v_cache, scale, pos, pos_dev, row_pos,
                                                     max_kv_len, window, q_weight, eps, norm_q, cos, sin,
                                                     chunk, out, workspace)
    c = args[13]
    kv_flags = (NORM_QK if norm_k else 0) | (ROPE if c is not None else 0) | (NORM_V if norm_v else 0)
    kw = _weight(k_weight, D) if norm_k else None
    need = lib().forge_attn_decode_workspace_bytes(args[0], B, T, q.shape[1], K, D, max_kv_len, chunk)
    zeroed, key = bool(workspace_zeroed), None
    if need and workspace is None and not torch.cuda.is_current_stream_capturing():
        (key, workspace), zeroed = _take_stream_workspace(dev, need), True
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace, zeroed = torch.empty(need, dtype=torch.uint8, device=dev), False
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    st = lib().forge_attn_decode_append(*args[:13], _ptr(k), k.stride(0), k.stride(1), k.stride(2),
                                        _ptr(v), v.stride(0), v.stride(1), v.stride(2), _ptr(kw), kv_flags,
                                        *args[13:], _ptr(workspace), ws_bytes, WS_ZEROED if zeroed else 0,
                                        _stream(dev))
    check(st, "forge_attn_decode_append")
    if key is not None:
        _put_back_stream_workspace(key, workspace)
    return out


def attn_decode_noalloc(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, scale: float,
                        out: torch.Tensor, pos: int | None = None, pos_dev: torch.Tensor | None = None,
                        row_pos: torch.Tensor | None = None, max_kv_len: int | None = None,
                        window: int = 0, q_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        norm_q: bool = False, cos: torch.Tensor | None = None,
                        sin: torch.Tensor | None = None, chunk: int = 0) -> torch.Tensor:
    """attn_decode through forge_attn_decode_noalloc: the split-K partials live in the
    library's own device array (at most NOALLOC_SCRATCH_BYTES), so the call allocates
    nothing on the device; `out` must be given. Calls that may overlap on one GPU race on
    that array."""
    args, out, dev, _, _ = _decode_args(q, k_cache, v_cache, scale, pos, pos_dev, row_pos, max_kv_len,
                                        window, q_weight, eps, norm_q, cos, sin, chunk, out, None)
    check(lib().forge_attn_decode_noalloc(*args, _stream(dev)), "forge_attn_decode_noalloc")
    return out


def attn_drafter(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                 n_past: int | None = None, n_past_dev: torch.Tensor | None = None,
                 window: int = 0, scale: float = 1.0, **kw) -> torch.Tensor:
    """The MTP drafter's attention onto the target's cache (sleuth/forge/infer/mtp.py:73-92,
    and its graph form with the position on the device, mtp.py:169-188): one query per
    row, at position n_past, over the n_past keys the target has stored (positions
    0 .. n_past-1); with a sliding window only keys k with n_past - k < window (llama.cpp's
    rule, mtp.py:84-86). Scale 1.0 by default. This is forge_attn_decode with the query
    placed at n_past - 1 (so it sees keys up to n_past - 1) and the window narrowed by
    one. q [B,H,1,D] (normalised and rotated by the drafter, or raw with norm_q/cos/sin
    as for attn_decode); returns [B,1,H,D]."""
    if q.shape[2] != 1:
        raise ValueError("the drafter attends with one query per row")
    if window < 0 or window == 1:
        raise ValueError("window must be 0 (global) or at least 2")
    w = window - 1 if window else 0
    if n_past_dev is not None:
        if n_past is not None:
            raise ValueError("give n_past or n_past_dev, not both")
        return attn_decode(q, k_cache, v_cache, scale=scale, pos_dev=n_past_dev.to(torch.int64) - 1,
                           window=w, **kw)
    if n_past is None or int(n_past) < 1:
        raise ValueError("n_past must be at least 1: the drafter needs keys the target stored")
    return attn_decode(q, k_cache, v_cache, scale=scale, pos=int(n_past) - 1, window=w, **kw)


PREFILL_HEAD_DIMS = (64, 128, 256, 512)


def _partials(need: int, dev: torch.device) -> torch.Tensor | None:
    """Workspace of a key-split prefill launch. None where it is not split, also for want of memory: the
    unsplit launch needs none."""
    try:
        return torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    except torch.OutOfMemoryError:
        return None


def prefill_supported(q: torch.Tensor) -> bool:
    return q.dtype in (torch.bfloat16, torch.float16) and q.shape[-1] in PREFILL_HEAD_DIMS


def attn_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float, offset: int = 0,
                 window: int = 0, q_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 norm_q: bool = False, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 doc_start: torch.Tensor | None = None, check_doc_start: bool = True) -> torch.Tensor:
    """Causal flash attention on MFMA: queries at positions offset..offset+T-1 over keys
    0..offset+T-1 of k/v [B,K,>=offset+T,D]. Returns [B,T,H,D].

    doc_start: [B, T] int32, the position of the first token of each query's document (the
    reference's document mask, transformer.py:271-275): query t also sees no key before it.
    It must be non-decreasing along T and at most the query's own position: checked here
    (two host synchronisations) unless check_doc_start is False, for a caller that built
    it so (the module's own starts, taken from the mask), or under graph capture."""
    if out is None and doc_start is None and q.dtype != torch.float32:
        r = host().prefill(q, k, v, float(scale), offset, window, q_weight, float(eps), bool(norm_q), cos, sin)
        if r is not None:
            return r if r.__class__ is not int else check(r, "forge_attn_prefill")
    B, H, T, D = q.shape
    Bk, K, S, Dk = k.shape
    if Bk != B or Dk != D or v.shape != k.shape or H % K:
        raise ValueError(f"q {tuple(q.shape)} does not fit k/v {tuple(k.shape)}")
    if S < offset + T:
        raise ValueError(f"k/v hold {S} positions, need offset + T = {offset + T}")
    if k.stride() != v.stride():
        raise ValueError("k and v must have the same strides")
    if not prefill_supported(q) or k.dtype != q.dtype:
        raise ValueError(f"MFMA prefill takes bf16/fp16 with head dim in {PREFILL_HEAD_DIMS}")
    dev = _need_device(q, k, v, cos, sin, out)
    _last_dim_contiguous(q, "q")
    _last_dim_contiguous(k, "k")
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    if s_b:
        raise ValueError("prefill takes [T, D] cos/sin shared by the batch")
    flags = (NORM_QK if norm_q else 0) | (ROPE if c is not None else 0)
    w = _weight(q_weight, D) if norm_q else None
    if out is None:
        out = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    elif out.shape != (B, T, H, D) or out.dtype != q.dtype:
        raise ValueError(f"out must be [B,T,H,D] = {(B, T, H, D)} {q.dtype}")
    doc_ptr, doc_stride = None, 0
    if doc_start is not None:
        if doc_start.dtype != torch.int32 or doc_start.shape != (B, T) or doc_start.device != dev:
            raise ValueError(f"doc_start must be int32 [B, T] = {(B, T)} on {dev}")
        if doc_start.stride(1) != 1:
            raise ValueError("doc_start: the last dimension must be contiguous")
        if check_doc_start and not torch.cuda.is_current_stream_capturing():
            pos = offset + torch.arange(T, device=dev, dtype=torch.int32)
            if bool(((doc_start < 0) | (doc_start > pos)).any()) or \
                    bool((doc_start[:, 1:] < doc_start[:, :-1]).any()):
                raise ValueError("doc_start must be non-decreasing and in [0, the query's position]")
        doc_ptr, doc_stride = _ptr(doc_start), doc_start.stride(0)
    # partials of a key-split launch (0: the shape is not split)
    need = 0 if doc_ptr else lib().forge_attn_prefill_workspace_bytes(dtype_code(q), B, T, H, K, D, int(offset), int(window))
    ws = _partials(need, dev)
    st = lib().forge_attn_prefill_ws(dtype_code(q), B, T, H, K, D, _ptr(q), q.stride(0), q.stride(1),
                                     q.stride(2), _ptr(w), float(eps), flags, _ptr(c), _ptr(s), s_t,
                                     _ptr(k), _ptr(v), k.stride(0), k.stride(1), k.stride(2),
                                     int(offset), int(window), float(scale), doc_ptr, doc_stride,
                                     _ptr(out), out.stride(0), out.stride(1), out.stride(2), _ptr(ws), need,
                                     _stream(dev))
    check(st, "forge_attn_prefill" if doc_start is None else "forge_attn_prefill_docs")
    return out


PREFILL_F32_HEAD_DIMS = (32, 64, 128)
# Keys from which the module takes fp32 prompts to attn_prefill_f32. Below, its error against 64 bits is
# up to 1.04 of the split-K path's (17 to 33 queries over at most 40 keys, means over 12 inputs);
# from 49 keys on it is 0.93 to 1.00 of it.
PREFILL_F32_MIN_KEYS = 49


def prefill_f32_supported(q: torch.Tensor, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                          q_weight: torch.Tensor | None = None, k: torch.Tensor | None = None, offset: int = 0) -> bool:
    """attn_prefill_f32 takes this q, these tables and this gain (16-byte aligned rows; attn_decode takes
    any), and keys k [B,K,S,D] of a slab whose rows up to a tile past the last query lie within 2^31
    bytes (attn_decode: the cache's own rows)."""
    _, _, T, D = q.shape
    if q.dtype is not torch.float32 or D not in PREFILL_F32_HEAD_DIMS:
        return False
    if k is not None and not D <= k.stride(2) < 2 ** 29 / (offset + T + 256):
        return False
    for t in (cos, sin, q_weight):
        if t is None:
            continue
        *rows, last = t.stride()
        if last != 1 or t.dtype is not torch.float32 or t.data_ptr() % 16 or (rows and (rows[0] % 4 or rows[-1] % 4)):
            return False   # (a gain, or tables of up to three dimensions)
    return True


def attn_prefill_f32(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float, offset: int = 0,
                     window: int = 0, q_weight: torch.Tensor | None = None, eps: float = 1e-6,
                     norm_q: bool = False, cos: torch.Tensor | None = None,
                     sin: torch.Tensor | None = None) -> torch.Tensor:
    """attn_prefill in fp32 (forge_attn_prefill_f32): queries at positions offset..offset+T-1 over
    keys 0..offset+T-1 of k/v [B,K,>=offset+T,D]. Returns [B,T,H,D]."""
    if q.dtype == torch.float32:
        r = host().prefill(q, k, v, float(scale), offset, window, q_weight, float(eps), bool(norm_q), cos, sin)
        if r is not None:
            return r if r.__class__ is not int else check(r, "forge_attn_prefill_f32")
    B, H, T, D = q.shape
    Bk, K, S, Dk = k.shape
    if Bk != B or Dk != D or v.shape != k.shape or H % K:
        raise ValueError(f"q {tuple(q.shape)} does not fit k/v {tuple(k.shape)}")
    if S < offset + T:
        raise ValueError(f"k/v hold {S} positions, need offset + T = {offset + T}")
    if k.stride() != v.stride():
        raise ValueError("k and v must have the same strides")
    if not prefill_f32_supported(q) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"fp32 prefill takes fp32 with head dim in {PREFILL_F32_HEAD_DIMS}")
    dev = _need_device(q, k, v, cos, sin)
    _last_dim_contiguous(q, "q")
    _last_dim_contiguous(k, "k")
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    if s_b:
        raise ValueError("prefill takes [T, D] cos/sin shared by the batch")
    flags = (NORM_QK if norm_q else 0) | (ROPE if c is not None else 0)
    w = _weight(q_weight, D) if norm_q else None
    out = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    need = lib().forge_attn_prefill_f32_workspace_bytes(B, T, H, K, D, int(offset), int(window))
    ws = _partials(need, dev)
    st = lib().forge_attn_prefill_f32(B, T, H, K, D, _ptr(q), q.stride(0), q.stride(1), q.stride(2), _ptr(w),
                                      float(eps), flags, _ptr(c), _ptr(s), s_t, _ptr(k), _ptr(v), k.stride(0),
                                      k.stride(1), k.stride(2), int(offset), int(window), float(scale), _ptr(out),
                                      out.stride(0), out.stride(1), out.stride(2), _ptr(ws), need, _stream(dev))
    check(st, "forge_attn_prefill_f32")
    return out


LINEAR_SMALL_ROWS = 16   # rows of x that forge_linear_small takes


def linear_small(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *,
                 w_up: torch.Tensor | None = None, gain: torch.Tensor | None = None, eps: float = 0.0,
                 norm: bool = False, residual: torch.Tensor | None = None) -> torch.Tensor | None:
    """F.linear(x, w, bias) of a decode or verify step (forge_linear_small), without autograd;
    norm: x gets RMSNorm (gain [K], fp32 or of x's type) first; w_up: silu(x . w^T) * (x . w_up^T); residual [..., N]:
    added to the result. None where the call is not of the kernel's form, or where torch's calls
    are faster (forge_linear_small_rows), for the caller to make those: it takes bf16/fp16 on one GPU, x [..., K] of at most 16 rows, K a multiple of
    32, everything contiguous and 16-byte aligned, and nothing (autocast, tracing, a dispatch or
    function mode, a tensor subclass, a forward-mode tangent) between the call and the memory."""
    if torch.is_autocast_enabled() or torch.compiler.is_compiling() or torch._C._get_tracing_state() is not None or \
            torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack():
        return None
    r = host().linear_small(x, w, bias, w_up, gain, float(eps), bool(norm), residual)
    return r if r.__class__ is not int else check(r, "forge_linear_small")


# ---------------------------------------------------------------- the paged cache, windows with sinks
# Partials of up to this many bytes stay with their stream (a decode or verify step's); a chunk's larger ones are
# allocated for the call
_PAGED_WS_KEPT = 32 << 20


class _PagedPartials:
    """The workspace of one attn_paged or attn_sinks call: the stream's cleared one (its counters are zero between
    calls), or memory for this call alone where it is large or a graph is being recorded (a graph keeps its own);
    None where nothing is split or memory is short."""

    def __init__(self, dev: torch.device, need: int):
        self.key, self.ws, self.need, self.flags = None, None, need, 0
        if need and need <= _PAGED_WS_KEPT and not torch.cuda.is_current_stream_capturing():
            self.key, self.ws = _take_stream_workspace(dev, need, _PAGED_WS)
            self.flags = WS_ZEROED
        elif need:
            self.ws = _partials(need, dev)

    def args(self) -> tuple:
        return _ptr(self.ws), 0 if self.ws is None else self.ws.numel(), self.flags

    def launched(self) -> None:
        if self.key is not None:
            _put_back_stream_workspace(self.key, self.ws, _PAGED_WS)


def _guard(dev: torch.device):
    """Launches go to the tensors' GPU, whichever is current."""
    return torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else contextlib.nullcontext()


def _aligned(t: torch.Tensor) -> bool:
    """16-byte aligned: the pointer and every stride of a dimension that has one (the last one contiguous)."""
    e = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and \
        all(st % e == 0 and st >= 0 for st, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def _strides3(t: torch.Tensor) -> tuple[int, int, int]:
    """The three leading strides, 0 where a dimension has one element (torch keeps any number there)."""
    return tuple(st if n > 1 else 0 for st, n in zip(t.stride()[:3], t.shape[:3]))


def _int32_rows(t: torch.Tensor | None, B: int, dev: torch.device, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != (B,) or t.device != dev:
        raise ValueError(f"{name} must be an int32 [B] tensor on {dev}")
    return t.contiguous()


def _pages(k_pages, v_pages, page_table, B: int, dev: torch.device):
    """Checks the pools [n_pages, K, page_size, D] and the table [B, max_pages]."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must be [n_pages, K, page_size, D]")
    n, _, size, _ = k_pages.shape
    if size < 16 or size & (size - 1) or n < 1:
        raise ValueError(f"pages hold a power of two of at least 16 positions, not {size}")
    if k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must have one dtype")
    if _strides3(k_pages) != _strides3(v_pages) or not _aligned(k_pages) or not _aligned(v_pages):
        raise ValueError("k_pages and v_pages must have the same strides, the last dimension contiguous, 16-byte aligned")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B or page_table.shape[1] < 1 or \
            page_table.device != dev:
        raise ValueError(f"page_table must be int32 [B, max_pages] with B={B} on {dev}")
    return page_table if page_table.stride(1) == 1 else page_table.contiguous()


def kv_append_paged(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, row_pos: torch.Tensor, *, new_lens: torch.Tensor | None = None,
                    k_weight: torch.Tensor | None = None, eps: float = 1e-6, norm_k: bool = False,
                    norm_v: bool = False, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None) -> None:
    """kv_append into a paged cache: k, v [B,K,T,D] get their norm and RoPE as there, and token t of row b goes to
    position row_pos[b] + t, i.e. slot position % page_size of page page_table[b, position // page_size] of the pools
    [n_pages, K, page_size, D]. Tokens t >= new_lens[b] (a padded batch) and positions without a page (an entry
    outside the pool, or past the table's end) are not written. Lengths, table and positions are int32 on the GPU. Rows
    may share the pages of a common prefix, but no two tokens of a call may go to one slot."""
    st = host().kv_append_paged(k, v, k_pages, v_pages, page_table, row_pos, new_lens, k_weight, float(eps), bool(norm_k),
                                bool(norm_v), cos, sin)
    if st is not None:
        return check(st, "forge_kv_append_paged")
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [B, K, T, D]")
    B, K, T, D = k.shape
    dev = _need_device(k, v, k_pages, v_pages, page_table, row_pos, new_lens, cos, sin, k_weight if norm_k else None)
    table = _pages(k_pages, v_pages, page_table, B, dev)
    if k_pages.shape[1] != K or k_pages.shape[3] != D:
        raise ValueError(f"pages {tuple(k_pages.shape)} do not fit new k {tuple(k.shape)}")
    e16 = 16 // k_pages.element_size()
    if D % (2 * e16) or D > 128 * e16:
        raise ValueError(f"head dim {D}: pages take multiples of {2 * e16} up to {128 * e16} in {k_pages.dtype}")
    k, v = (x if x.dtype == k_pages.dtype and _aligned(x) else x.to(k_pages.dtype).clone(memory_format=torch.contiguous_format)
            for x in (k, v))
    rp, nl = _int32_rows(row_pos, B, dev, "row_pos"), _int32_rows(new_lens, B, dev, "new_lens")
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    flags = (NORM_QK if norm_k else 0) | (ROPE if c is not None else 0) | (NORM_V if norm_v else 0)
    w = _weight(k_weight, D) if norm_k else None
    with _guard(dev):
        st = lib().forge_kv_append_paged(dtype_code(k_pages), B, T, K, D, _ptr(k), *_strides3(k), _ptr(v), *_strides3(v),
                                         _ptr(k_pages), _ptr(v_pages), *_strides3(k_pages), k_pages.shape[0],
                                         k_pages.shape[2], _ptr(table), table.stride(0) if B > 1 else 0, table.shape[1],
                                         _ptr(rp), _ptr(nl), _ptr(w), float(eps), flags, _ptr(c), _ptr(s), s_b, s_t,
                                         _stream(dev))
    check(st, "forge_kv_append_paged")


def paged_supported(dtype: torch.dtype, D: int) -> bool:
    """attn_paged and attn_sinks take this dtype and head dim."""
    return dtype in _DTYPES and (D in (32, 64, 128, 256) or (D == 512 and dtype != torch.float32))


def _new_token_args(q, cache, scale, q_weight, eps, norm_q, cos, sin, window, sinks, out):
    """Checks what attn_paged and attn_sinks share; (q, C arguments from dtype to s_cos_t, out)."""
    if not 1e-37 <= float(scale) <= 1e38:
        raise ValueError(f"scale must be positive and finite, not {scale}")
    if q.dim() != 4 or q.shape[1] % cache.shape[1] or q.shape[3] != cache.shape[3]:
        raise ValueError(f"q {tuple(q.shape)} does not fit the cache {tuple(cache.shape)}")
    B, H, T, D = q.shape
    if q.dtype != cache.dtype:
        raise ValueError(f"q is {q.dtype} but the cache is {cache.dtype}")
    if not paged_supported(q.dtype, D):
        raise ValueError(f"head dim {D} in {q.dtype}: 32, 64, 128, 256, and 512 in 16 bits")
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError("window and sinks must not be negative, and sinks need a window")
    if max(window, sinks) >= 1 << 30:
        raise ValueError("window and sinks must be below 2^30 (a window of 0 sees every key)")
    dev = q.device
    if not _aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    elif out.shape != (B, T, H, D) or out.dtype != q.dtype or out.device != dev or not _aligned(out) or \
            any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape)):
        raise ValueError(f"out must be a 16-byte aligned [B,T,H,D] = {(B, T, H, D)} {q.dtype} on {dev}")
    c, s, s_b, s_t = _rope_tables(cos, sin, B, T, D)
    w = _weight(q_weight, D) if norm_q else None
    if w is not None and w.data_ptr() % 16:
        w = w.clone()
    flags = (NORM_QK if norm_q else 0) | (ROPE if c is not None else 0)
    keep = (q, w, c, s)   # alive until the launch
    return keep, (dtype_code(q), B, T, H, cache.shape[1], D, _ptr(q), *_strides3(q), _ptr(w), float(eps), flags, _ptr(c),
                  _ptr(s), s_b, s_t), out


def attn_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               row_pos: torch.Tensor, *, scale: float, new_lens: torch.Tensor | None = None,
               max_kv_len: int | None = None, window: int = 0, sinks: int = 0, q_weight: torch.Tensor | None = None,
               eps: float = 1e-6, norm_q: bool = False, cos: torch.Tensor | None = None,
               sin: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens q [B,H,T,D] over the paged cache (kv_append_paged), which holds their keys
    already: one token per row or a chunk of thousands, rows of any lengths. Query t of row b sits at
    p = row_pos[b] + t and sees keys s <= p; with a window those with s > p - window, and the first `sinks` positions.
    Keys whose table entry lies outside the pool (-1: given back) are invisible. Returns [B,T,H,D]; rows
    t >= new_lens[b] and rows that see nothing are zeros. max_kv_len: an upper bound on row_pos[b] + new_lens[b]
    (default: what the table can hold); it sizes the launch."""
    if out is None:
        r = host().attn_paged(_PAGED_WS, q, k_pages, v_pages, page_table, row_pos, new_lens, float(scale), max_kv_len, window, sinks,
                              q_weight, float(eps), bool(norm_q), cos, sin)
        if r is not None:
            return r if r.__class__ is not int else check(r, "forge_attn_paged")
    dev = _need_device(q, k_pages, v_pages, page_table, row_pos, new_lens, cos, sin, q_weight if norm_q else None, out)
    if q.dim() != 4:
        raise ValueError(f"q {tuple(q.shape)} must be [B, H, T, D]")
    B, T = q.shape[0], q.shape[2]
    table = _pages(k_pages, v_pages, page_table, B, dev)
    rp, nl = _int32_rows(row_pos, B, dev, "row_pos"), _int32_rows(new_lens, B, dev, "new_lens")
    size = k_pages.shape[2]
    most = table.shape[1] * size
    max_kv_len = most if max_kv_len is None else min(int(max_kv_len), most)
    if max_kv_len < 1:
        raise ValueError("max_kv_len must be positive")
    keep, args, out = _new_token_args(q, k_pages, scale, q_weight, eps, norm_q, cos, sin, window, sinks, out)
    with _guard(dev):
        ws = _PagedPartials(dev, lib().forge_attn_paged_workspace_bytes(*args[:6], max_kv_len, int(window), int(sinks)))
        st = lib().forge_attn_paged(*args, _ptr(k_pages), _ptr(v_pages), *_strides3(k_pages), k_pages.shape[0], size,
                                    _ptr(table), table.stride(0) if B > 1 else 0, table.shape[1], _ptr(rp), _ptr(nl),
                                    max_kv_len, int(window), int(sinks), float(scale), _ptr(out), *_strides3(out),
                                    *ws.args(), _stream(dev))
    check(st, "forge_attn_paged")
    ws.launched()
    return out


def attn_sinks(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, scale: float, window: int,
               sinks: int, pos: int | None = None, pos_dev: torch.Tensor | None = None,
               row_pos: torch.Tensor | None = None, max_kv_len: int | None = None,
               q_weight: torch.Tensor | None = None, eps: float = 1e-6, norm_q: bool = False,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               out: torch.Tensor | None = None, fixed_cut: bool = False) -> torch.Tensor:
    """Sliding-window attention whose first `sinks` positions stay visible, over a contiguous cache
    [B,K,max_len,D] that holds the new keys already: query t of row b sits at p = base_b + t (row_pos, pos_dev or
    pos, as attn_decode) and sees keys s <= p with s > p - window or s < sinks. Any T: whole prompts, chunks, verify and
    decode steps. Returns [B,T,H,D].

    fixed_cut (T <= 16): a token's result is the same, bit for bit, in every such call on caches of one shape, whatever T,
    max_kv_len and the way the position is given: a verify step's rows equal the decodes of its tokens."""
    fixed_cut = bool(fixed_cut)
    if out is None:
        r = host().attn_sinks(_PAGED_WS, q, k_cache, v_cache, float(scale), window, sinks, pos, pos_dev, row_pos, max_kv_len, q_weight,
                              float(eps), bool(norm_q), cos, sin, fixed_cut)
        if r is not None:
            return r if r.__class__ is not int else check(r, "forge_attn_sinks")
    dev = _need_device(q, k_cache, v_cache, pos_dev, row_pos, cos, sin, q_weight if norm_q else None, out)
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or k_cache.dtype != v_cache.dtype or \
            q.dim() != 4 or q.shape[0] != k_cache.shape[0]:
        raise ValueError(f"q {tuple(q.shape)} does not fit caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if _strides3(k_cache) != _strides3(v_cache) or not _aligned(k_cache) or not _aligned(v_cache):
        raise ValueError("k and v caches must have the same strides, the last dimension contiguous, 16-byte aligned")
    if window < 1:
        raise ValueError("attn_sinks needs a window (attn_decode and attn_prefill see every key)")
    B, T, max_len = q.shape[0], q.shape[2], k_cache.shape[2]
    if fixed_cut and T > DECODE_CHUNK_MAX_T:
        raise ValueError(f"fixed_cut is for steps of at most {DECODE_CHUNK_MAX_T} tokens")
    rp, pd, p0 = _positions(pos, pos_dev, row_pos, B, dev)
    if rp is None and pd is None:
        if not 0 <= p0 <= max_len - T:
            raise ValueError(f"pos {p0} + {T} tokens do not fit a cache of {max_len}")
        max_kv_len = p0 + T
    max_kv_len = max_len if max_kv_len is None else min(int(max_kv_len), max_len)
    if max_kv_len < 1:
        if B == 0 or T == 0:
            max_kv_len = 1
        else:
            raise ValueError("max_kv_len must be positive")
    keep, args, out = _new_token_args(q, k_cache, scale, q_weight, eps, norm_q, cos, sin, window, sinks, out)
    with _guard(dev):
        need = lib().forge_attn_sinks_fixed_workspace_bytes(*args[:6], max_len, int(window), int(sinks)) if fixed_cut else \
            lib().forge_attn_sinks_workspace_bytes(*args[:6], max_kv_len, int(window), int(sinks))
        if fixed_cut:
            args = (*args[:12], args[12] | FIXED_CUT, *args[13:])
        ws = _PagedPartials(dev, need)
        if fixed_cut and need and ws.ws is None:   # (unsplit, its bits would be others)
            raise torch.cuda.OutOfMemoryError(f"attn_sinks: no memory for {need} bytes of partials, which fixed_cut needs")
        st = lib().forge_attn_sinks(*args, _ptr(k_cache), _ptr(v_cache), *_cache_strides(k_cache), max_len, _ptr(rp), _ptr(pd),
                                    p0, max_kv_len, int(window), int(sinks), float(scale), _ptr(out), *_strides3(out),
                                    *ws.args(), _stream(dev))
    check(st, "forge_attn_sinks")
    ws.launched()
    return out


def _cache_strides(t: torch.Tensor) -> tuple[int, int, int]:
    """_strides3 with a positions' stride the kernels accept where there is one position."""
    b, h, s = _strides3(t)
    return b, h, s or t.shape[3]


__all__ = ["head_norm_rope", "kv_append", "attn_decode", "attn_decode_append", "attn_decode_noalloc", "attn_prefill", "attn_prefill_f32", "decode_chunk",
           "decode_workspace_bytes", "attn_drafter", "prefill_supported", "kv_append_paged",
           "attn_paged", "attn_sinks", "paged_supported", "dtype_code", "_lib"]
