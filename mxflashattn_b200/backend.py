"""The single CUDA backend behind ``dispatch``: torch tensors -> libmxfa_b200.

It exposes the extension contract the reference's dispatcher calls
(``getattr(ext, operation)(*extension_args)`` guarded by ``is_available()``,
mxflashattn/dispatch.py:131-137) with the positional argument lists the
reference's public API builds (mxflashattn/api.py:53, :122-133, :251-262):

* ``flash_attn_func(q, k, v, causal, scale)``
* ``flash_attn_varlen_func(q, k, v, cu_q, cu_k, max_q, max_k, causal, scale)``
* ``flash_attn_with_kvcache(q, k_cache, v_cache, k, v, cache_seqlens, block_table, scale, causal)``

PyTorch is used for device buffers and the current stream only; all math
runs in the sm_100a kernels.  Every call is asynchronous on the current
stream and reads nothing back to the host.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16)


# torch's own unwrapped queries of the current device and stream: a tenth of the time of the public
# functions, which build a context check or a Stream object around them
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)

_AVAILABLE: dict[int, bool] = {}


_CUDA_OK: list[bool] = []


def is_available() -> bool:
    """True when the current CUDA device is sm_100 and the library is usable (cached per device)."""
    if not _CUDA_OK:
        if not torch.cuda.is_available():
            return False
        _CUDA_OK.append(True)
    dev = _current_device()
    cached = _AVAILABLE.get(dev)
    if cached is not None:
        return cached
    try:
        ok = bool(_L().mxfa_is_available())
    except _lib.NativeLibraryError:
        ok = False
    _AVAILABLE[dev] = ok
    return ok


def _bf16(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return 1
    if t.dtype == torch.float16:
        return 0
    raise TypeError(f"the CUDA backend supports float16 and bfloat16, got {t.dtype}")


def _i32(t: torch.Tensor) -> torch.Tensor:
    return t if (t.dtype == torch.int32 and t.is_contiguous()) else t.to(torch.int32).contiguous()


def _contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


_NULL_CTX = contextlib.nullcontext()


def _on(t: torch.Tensor):
    """Device context for a launch: a no-op when ``t`` already lives on the current device."""
    idx = t.device.index
    return _NULL_CTX if idx == _current_device() else torch.cuda.device(idx)


_LIB: list = []


def _L():
    """The loaded library (cached)."""
    if not _LIB:
        _LIB.append(_lib.load())
    return _LIB[0]


def _stream(t: torch.Tensor) -> int:
    return _raw_stream(t.device.index)


# ------------------------------------------------------------------ prefill

def flash_attn_varlen_func(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, causal,
                           softmax_scale, *, return_lse: bool = False, exact_p: bool = False):
    """Packed varlen forward: q [Tq, HQ, D], k/v [Tk, HKV, D] -> out [Tq, HQ, D].

    ``exact_p``: keep P at ~16 significant bits in the P.V product
    (``mxfa_varlen_fwd_exact_launch``, 1.5x the tensor work) instead of
    rounding it once to the input type.
    """
    q, k, v = _contig(q), _contig(k), _contig(v)
    out = torch.empty_like(q)
    lse = torch.empty((q.shape[0], q.shape[1]), device=q.device, dtype=torch.float32) if return_lse else None
    cu_q, cu_k = _i32(cu_seqlens_q), _i32(cu_seqlens_k)
    batch = cu_q.numel() - 1
    name = "mxfa_varlen_fwd_exact_launch" if exact_p else "mxfa_varlen_fwd_launch"
    with _on(q):
        rc = getattr(_L(), name)(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(),
            _lib.ptr(lse), batch, int(max_seqlen_q), int(max_seqlen_k), q.shape[0], k.shape[0], q.shape[1],
            k.shape[1], q.shape[2], int(bool(causal)), _bf16(q), float(softmax_scale), _stream(q))
    _lib.check(rc, name)
    return (out, lse) if return_lse else out


def flash_attn_func(q, k, v, causal, softmax_scale, *, return_lse: bool = False, exact_p: bool = False):
    """Dense batched forward: q [B, Sq, HQ, D], k/v [B, Sk, HKV, D] -> out [B, Sq, HQ, D]."""
    q, k, v = _contig(q), _contig(k), _contig(v)
    out = torch.empty_like(q)
    B, Sq, HQ, D = q.shape
    lse = torch.empty((B, Sq, HQ), device=q.device, dtype=torch.float32) if return_lse else None
    name = "mxfa_varlen_fwd_exact_launch" if exact_p else "mxfa_varlen_fwd_launch"
    with _on(q):
        rc = getattr(_L(), name)(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), None, None, out.data_ptr(), _lib.ptr(lse), B, Sq,
            k.shape[1], B * Sq, B * k.shape[1], HQ, k.shape[2], D, int(bool(causal)), _bf16(q),
            float(softmax_scale), _stream(q))
    _lib.check(rc, name)
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ decode

_PLANS: dict[tuple, tuple[int, int]] = {}
_PLANS_KEPT = 4096  # a serving loop may ask for another length every step


def kvcache_plan(batch: int, q_len: int, q_heads: int, kv_heads: int, head_dim: int, max_len: int):
    """(num_splits, chunk_len) the library picks for this shape on the current device (cached, the latest ones)."""
    key = (_current_device() if (_CUDA_OK or torch.cuda.is_available()) else -1, batch, q_len, q_heads,
           kv_heads, head_dim, max_len)
    plan = _PLANS.get(key)
    if plan is None:
        np_, cl = ctypes.c_int(0), ctypes.c_int(0)
        _lib.check(_L().mxfa_kvcache_plan(batch, q_len, q_heads, kv_heads, head_dim, max_len,
                                                  ctypes.byref(np_), ctypes.byref(cl)), "mxfa_kvcache_plan")
        if len(_PLANS) >= _PLANS_KEPT:
            _PLANS.clear()
        plan = _PLANS[key] = (int(np_.value), int(cl.value))
    return plan


_COUNTERS: dict[tuple, "torch.Tensor"] = {}
_CAPTURE_COUNTERS: dict[tuple, tuple[int, "torch.Tensor"]] = {}


def _capture_id(device, stream_handle: int) -> int:
    """Id of the graph capture that the stream is part of (ids are never used twice), 0 without one."""
    if device.type != "cuda" or not _capturing():
        return 0
    out = ctypes.c_ulonglong(0)
    _lib.check(_L().mxfa_stream_capture_id(stream_handle, ctypes.byref(out)), "mxfa_stream_capture_id")
    return int(out.value)


def split_counters(device, stream_handle: int, nbytes: int):
    """Zeroed counter array for single-launch splits on one (device, stream).

    Every counted launch leaves its counters at zero again, so one array per
    stream is reused by all launches ordered on that stream; it only grows.

    A captured launch replays on any stream, next to other graphs and to eager
    launches, so a graph shares its counters with nobody: the first launch of a
    capture allocates them in the graph's own memory, and their zeroing is a
    node of that graph, which the launches captured after it follow.
    """
    key = (device, stream_handle)
    n = max(nbytes // 4, 1)
    capture = _capture_id(device, stream_handle)
    if capture:
        # kept until the stream's next capture: while this one runs, nothing else may get the memory
        held, buf = _CAPTURE_COUNTERS.get(key, (0, None))
        if held != capture or buf.numel() < n:
            buf = torch.zeros((max(n, 4096),), device=device, dtype=torch.int32)
            _CAPTURE_COUNTERS[key] = (capture, buf)
        return buf
    buf = _COUNTERS.get(key)
    if buf is None or buf.numel() < n:
        buf = _COUNTERS[key] = torch.zeros((max(n, 4096),), device=device, dtype=torch.int32)
    return buf


def kvcache_length_order(cache_seqlens):
    """Longest-first order of the batch (int32 [B]: order[rank] = sequence), for ``length_order=``.

    Computed on the device (``mxfa_kvcache_length_order_launch``) once per
    step and passed to every layer's ``kvcache_attention``, it replaces the
    ranking each CTA otherwise does on every layer.  Batches of one or of more
    than 512 sequences need none (None is returned)."""
    seq = _i32(cache_seqlens)
    B = seq.shape[0]
    if B <= 1 or B > 512:
        return None
    order = torch.empty((B,), device=seq.device, dtype=torch.int32)
    with _on(seq):
        rc = _L().mxfa_kvcache_length_order_launch(seq.data_ptr(), B, order.data_ptr(), _stream(seq))
    _lib.check(rc, "mxfa_kvcache_length_order_launch")
    return order


def kvcache_attention(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, causal, *,
                      append_len: int = 0, return_lse: bool = False, num_splits: int = 0, chunk_len: int = 0,
                      out=None, k_new=None, v_new=None, single_launch: bool = True, k_scale: float = 1.0,
                      v_scale: float = 1.0, length_order=None):
    """Attention of q [B, Sq, HQ, D] over the cached tokens (+ ``append_len``).

    ``cache_seqlens`` holds the lengths before the append.  Without
    ``k_new``/``v_new`` nothing is written to the caches (the appended rows
    must already be there); with them the same launch writes those rows into
    the caches first (``mxfa_kvcache_append_attention_launch``).
    ``num_splits``/``chunk_len`` 0 = library plan.  A split plan runs as one
    launch (the last split CTA of each unit merges) unless ``single_launch``
    is False, which keeps the separate combine kernel.  ``torch.float8_e4m3fn``
    caches attend to ``k_cache * k_scale`` and ``v_cache * v_scale``.
    ``length_order`` (from ``kvcache_length_order``) schedules the sequences
    without the per-CTA ranking; it is ignored by the fused append.
    """
    B, Sq, HQ, D = q.shape
    q = _contig(q)
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the CUDA backend requires contiguous k_cache / v_cache")
    seq = _i32(cache_seqlens)
    bt = None if block_table is None else _i32(block_table)
    PS = k_cache.shape[1]
    HKV = k_cache.shape[2]
    if bt is not None:
        btw, pages = bt.shape[1], k_cache.shape[0]
        max_len = btw * PS
    else:
        btw, pages = 0, k_cache.shape[0]
        max_len = PS
    if out is None:
        out = torch.empty_like(q)
    lse = torch.empty((B, Sq, HQ), device=q.device, dtype=torch.float32) if return_lse else None
    lib = _L()
    if num_splits <= 0 or chunk_len <= 0:
        num_splits, chunk_len = kvcache_plan(B, Sq, HQ, HKV, D, max_len)
    ws = None
    ws_bytes = 0
    if num_splits > 1:
        ws_bytes = int(lib.mxfa_split_workspace_bytes(B * Sq * HQ, D, num_splits))
        ws = torch.empty((ws_bytes // 4,), device=q.device, dtype=torch.float32)
    with _on(q):
        stream = _stream(q)
        counters = None
        if num_splits > 1 and single_launch:
            counters = split_counters(q.device, stream, int(lib.mxfa_split_counter_bytes(B, Sq, HQ, HKV)))
        if length_order is not None and k_new is None:
            order = _i32(length_order)
            if order.shape != (B,) or order.device != q.device:
                raise ValueError(f"length_order must be int32 [{B}] on {q.device}")
            fp8 = _is_fp8(k_cache)
            name = "mxfa_kvcache_attention_ordered_launch"
            rc = lib.mxfa_kvcache_attention_ordered_launch(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(), order.data_ptr(),
                out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, _lib.ptr(counters), B, Sq, HQ, HKV, D, PS,
                btw, pages, int(append_len), num_splits, chunk_len, int(bool(causal)), _bf16(q),
                float(softmax_scale), int(fp8), float(k_scale), float(v_scale), stream)
        elif _is_fp8(k_cache):
            if k_new is not None:
                raise ValueError("the fused append does not take float8_e4m3fn rows; append with kv_append first")
            name = "mxfa_kvcache_attention_fp8_launch"
            rc = lib.mxfa_kvcache_attention_fp8_launch(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(),
                out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, _lib.ptr(counters), B, Sq, HQ, HKV, D, PS,
                btw, pages, int(append_len), num_splits, chunk_len, int(bool(causal)), _bf16(q),
                float(softmax_scale), float(k_scale), float(v_scale), stream)
        elif k_new is None:
            if counters is None:
                name = "mxfa_kvcache_attention_launch"
                rc = lib.mxfa_kvcache_attention_launch(
                    q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(),
                    out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, B, Sq, HQ, HKV, D, PS, btw, pages,
                    int(append_len), num_splits, chunk_len, int(bool(causal)), _bf16(q), float(softmax_scale),
                    stream)
            else:
                name = "mxfa_kvcache_attention_counted_launch"
                rc = lib.mxfa_kvcache_attention_counted_launch(
                    q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(),
                    out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, counters.data_ptr(), B, Sq, HQ, HKV,
                    D, PS, btw, pages, int(append_len), num_splits, chunk_len, int(bool(causal)), _bf16(q),
                    float(softmax_scale), stream)
        else:
            name = "mxfa_kvcache_append_attention_launch"
            k_new, v_new = _contig(k_new), _contig(v_new)
            rc = lib.mxfa_kvcache_append_attention_launch(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(),
                out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, _lib.ptr(counters), k_new.data_ptr(),
                v_new.data_ptr(), B, Sq, HQ, HKV, D, PS, btw, pages, int(k_new.shape[1]), num_splits, chunk_len,
                int(bool(causal)), _bf16(q), float(softmax_scale), stream)
    _lib.check(rc, name)
    return (out, lse) if return_lse else out


def _is_fp8(t) -> bool:
    return t.dtype == getattr(torch, "float8_e4m3fn", None)


def fused_append_supported(q, k_cache, k) -> bool:
    """True when one launch can append ``k``/``v`` and attend (up to 16 query rows per KV head)."""
    B, Sq, HQ, D = q.shape
    HKV = k_cache.shape[2]
    return (k is not None and k.shape[1] > 0 and HQ % HKV == 0 and Sq * (HQ // HKV) <= 16
            and k.dtype == k_cache.dtype and not _is_fp8(k_cache))


def kv_append(k_cache, v_cache, k, v, cache_seqlens, block_table) -> None:
    """Write k/v [B, Sk, HKV, D] at positions cache_seqlens[b] + i (no length update)."""
    k, v = _contig(k), _contig(v)
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the CUDA backend requires contiguous k_cache / v_cache")
    seq = _i32(cache_seqlens)
    bt = None if block_table is None else _i32(block_table)
    B, Sk, HKV, D = k.shape
    with _on(k):
        rc = _L().mxfa_kv_append_launch(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(), B,
            Sk, HKV, D, k_cache.shape[1], 0 if bt is None else bt.shape[1], k_cache.shape[0], k.element_size(),
            _stream(k))
    _lib.check(rc, "mxfa_kv_append_launch")


def seqlens_add_(cache_seqlens: torch.Tensor, delta: int) -> None:
    """In-place ``cache_seqlens += delta`` on the device (int32 or int64)."""
    if cache_seqlens.dtype not in (torch.int32, torch.int64) or not cache_seqlens.is_contiguous():
        cache_seqlens.add_(delta)
        return
    with _on(cache_seqlens):
        rc = _L().mxfa_seqlens_add_launch(
            cache_seqlens.data_ptr(), int(cache_seqlens.dtype == torch.int64), cache_seqlens.numel(), int(delta),
            _stream(cache_seqlens))
    _lib.check(rc, "mxfa_seqlens_add_launch")


def flash_attn_with_kvcache(q, k_cache, v_cache, k, v, cache_seqlens, block_table, softmax_scale, causal,
                            k_scale: float = 1.0, v_scale: float = 1.0, out=None, length_order=None):
    """``flash_attn_with_kvcache`` semantics of the reference (reference.py:88-139).

    Appends ``k``/``v`` (when given) at the current lengths, attends over the
    grown cache, then advances ``cache_seqlens`` in place -- all on the
    current stream, with no host synchronisation.  ``out`` (optional, q's
    shape and dtype, contiguous) receives the result.  ``length_order``
    (optional, from ``kvcache_length_order``) schedules the sequences without
    the per-launch ranking.
    """
    if q.shape[1] == 0:
        if k is not None:
            kv_append(k_cache, v_cache, k, v, cache_seqlens, block_table)
            seqlens_add_(cache_seqlens, k.shape[1])
        return out if out is not None else torch.empty_like(q)
    append_len = 0
    if k is not None and fused_append_supported(q, k_cache, k):
        # decode shapes: the attention kernel writes the new rows itself (one launch fewer)
        append_len = k.shape[1]
        out = kvcache_attention(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, causal,
                                append_len=append_len, k_new=k, v_new=v, out=out)
        seqlens_add_(cache_seqlens, append_len)
        return out
    if k is not None:
        kv_append(k_cache, v_cache, k, v, cache_seqlens, block_table)
        append_len = k.shape[1]
    out = kvcache_attention(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, causal,
                            append_len=append_len, k_scale=k_scale, v_scale=v_scale, out=out,
                            length_order=length_order)
    if k is not None:
        seqlens_add_(cache_seqlens, append_len)
    return out


def kvcache_attention_packed(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, *,
                             num_splits: int = 0, chunk_len: int = 0, out=None):
    """Local half of a context-split decode: packed f32 [B*HQ, D+1] = (normalised O, LSE) per row."""
    B, Sq, HQ, D = q.shape
    if Sq != 1:
        raise ValueError("packed local attention takes one query token per sequence")
    q = _contig(q)
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the CUDA backend requires contiguous k_cache / v_cache")
    seq = _i32(cache_seqlens)
    bt = None if block_table is None else _i32(block_table)
    PS, HKV = k_cache.shape[1], k_cache.shape[2]
    btw = 0 if bt is None else bt.shape[1]
    max_len = btw * PS if bt is not None else PS
    if num_splits <= 0 or chunk_len <= 0:
        num_splits, chunk_len = kvcache_plan(B, 1, HQ, HKV, D, max_len)
    lib = _L()
    ws_bytes = int(lib.mxfa_split_workspace_bytes(B * HQ, D, num_splits))
    ws = torch.empty((max(ws_bytes, 16) // 4,), device=q.device, dtype=torch.float32)
    if out is None:
        out = torch.empty((B * HQ, D + 1), device=q.device, dtype=torch.float32)
    with _on(q):
        rc = lib.mxfa_kvcache_attention_packed_launch(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(bt), seq.data_ptr(), out.data_ptr(),
            ws.data_ptr(), ws_bytes, B, HQ, HKV, D, PS, btw, k_cache.shape[0], num_splits, chunk_len, _bf16(q),
            float(softmax_scale), _stream(q))
    _lib.check(rc, "mxfa_kvcache_attention_packed_launch")
    return out


# ------------------------------------ a ragged batch over a paged cache

def _rows16(t):
    """``t`` with unit stride along D and 16-byte rows: itself, or a packed copy."""
    s = t.stride()
    if s[2] == 1 and s[0] and s[1] and s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def kvcache_append_varlen(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, k_scales, v_scales) -> None:
    """Packed k/v [T, HKV, D] into their pages, copied or quantised (no length update)."""
    k = k if k.stride(2) == 1 else k.contiguous()
    v = v if v.stride(2) == 1 else v.contiguous()
    cu, seq, bt = _i32(cu_seqlens), _i32(cache_seqlens), _i32(block_table)
    T, HKV, D = k.shape
    ks, vs = k.stride(), v.stride()
    with _on(k):
        rc = _L().mxfa_kvcache_append_varlen_launch(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scales),
            _lib.ptr(v_scales), cu.data_ptr(), seq.data_ptr(), bt.data_ptr(), T, seq.shape[0], HKV, D,
            k_cache.shape[1], bt.shape[1], k_cache.shape[0], ks[0], ks[1], vs[0], vs[1], _bf16(k), _stream(k))
    _lib.check(rc, "mxfa_kvcache_append_varlen_launch")


def kvcache_gather_varlen(k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, k_scales, v_scales, k, v) -> None:
    """Packed k/v [T, HKV, D] (written) from their pages."""
    cu, seq, bt = _i32(cu_seqlens), _i32(cache_seqlens), _i32(block_table)
    T, HKV, D = k.shape
    with _on(k):
        rc = _L().mxfa_kvcache_gather_varlen_launch(
            k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scales), _lib.ptr(v_scales), cu.data_ptr(),
            seq.data_ptr(), bt.data_ptr(), k.data_ptr(), v.data_ptr(), T, seq.shape[0], HKV, D, k_cache.shape[1],
            bt.shape[1], k_cache.shape[0], _bf16(k), _stream(k))
    _lib.check(rc, "mxfa_kvcache_gather_varlen_launch")


_SCRATCH: dict[tuple, "torch.Tensor"] = {}
_SCRATCH_KEEP = 64 << 20


def _scratch(q, stream_handle: int, nbytes: int):
    """Workspace for launches ordered on one (device, stream): kept and grown up to 64 MB, larger ones per call.

    Nothing in it outlives the launch that writes it, so launches ordered on
    the stream share it, as they share the split counters.
    """
    # a captured launch replays with the pointer it was given: its workspace belongs to the graph
    if nbytes > _SCRATCH_KEEP or (q.is_cuda and _capturing()):
        return q.new_empty((nbytes,), dtype=torch.uint8)
    key = (q.device, stream_handle)
    buf = _SCRATCH.get(key)
    if buf is None or buf.shape[0] < nbytes:
        buf = _SCRATCH[key] = q.new_empty((nbytes,), dtype=torch.uint8)
    return buf


_CHUNK_SIZES: dict[tuple, tuple[int, int]] = {}


def _chunk_sizes(kv_heads: int, head_dim: int) -> tuple[int, int]:
    """(workspace bytes, counter bytes) of the tiled attention on the current device (cached)."""
    key = (_current_device() if (_CUDA_OK or torch.cuda.is_available()) else -1, kv_heads, head_dim)
    sizes = _CHUNK_SIZES.get(key)
    if sizes is None:
        lib = _L()
        sizes = _CHUNK_SIZES[key] = (int(lib.mxfa_chunk_workspace_bytes(kv_heads, head_dim)),
                                     int(lib.mxfa_chunk_counter_bytes(kv_heads)))
    return sizes


# Unpacking costs a pass over the cached rows and then runs the faster 16-bit kernel; converting in the
# kernel repeats its work for every tile of a sequence. Device us, converted / unpacked, bf16, 8 KV heads, 4 heads each:
#   one sequence of 15,360 cached tokens: 32 new ones (1 tile) 65 / 76, 64 (2) 60 / 64, 96 (3) 67 / 65,
#     128 (4) 80 / 68, 256 (8) 133 / 93, 1,024 (32) 468 / 248
#   8 sequences of 2,000: 64 each 43 / 51, 128 (4) 81 / 71, 256 159 / 122
#   512 tokens on 4,096 and 31 decodes on as many (2 tiles a sequence): 207 / 251
# fp16 (with the converting launch behind): 128 on 15,360 84 / 75, 8 x 128 on 2,000 83 / 85, 1,024 495 / 262.
# bf16 P is rounded to 8 bits on unpacked rows, as on a 16-bit cache, and to f16's 11 in the converting kernel.
UNPACK_TILES = 4
UNPACK_BYTES = 1 << 30
UNPACK_BATCH = 65535  # sequences of one unpacking launch


def unpack_pays(total_q: int, batch: int, group: int, kv_heads: int, head_dim: int, max_len: int) -> bool:
    """Whether a quantised call first unpacks its sequences to 16 bits."""
    return (total_q * group >= UNPACK_TILES * 128 * batch and max_len > 0  # (empty caches have no rows to unpack)
            and batch <= UNPACK_BATCH and 4 * batch * max_len * kv_heads * head_dim <= UNPACK_BYTES)


_MAX_GROUP = 128  # query heads of one KV head that the tiled kernel takes
_MAX_STEP_BATCH = 65535  # sequences that the split-KV kernel takes


def kvcache_chunk_plan(cu_seqlens_q, cache_seqlens, total_q: int, q_heads: int, kv_heads: int, causal: bool):
    """The items of a step's ragged attention (int32, on the device), or None where no tiled call needs them."""
    B = cache_seqlens.numel()
    if total_q == 0 or B == 0 or q_heads // kv_heads > _MAX_GROUP:
        return None
    cu, seq = _i32(cu_seqlens_q), _i32(cache_seqlens)
    lib = _L()
    with _on(cu):
        nbytes = int(lib.mxfa_chunk_plan_bytes(total_q, B, q_heads, kv_heads))
        table = torch.empty((nbytes // 4,), device=cu.device, dtype=torch.int32)
        rc = lib.mxfa_kvcache_chunk_plan_launch(cu.data_ptr(), seq.data_ptr(), table.data_ptr(), nbytes, total_q, B,
                                                q_heads, kv_heads, int(causal), _stream(cu))
    _lib.check(rc, "mxfa_kvcache_chunk_plan_launch")
    return table


def flash_attn_varlen_with_kvcache(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, max_seqlen_q,
                                   max_seqlen_k, softmax_scale, causal, k_scales=None, v_scales=None, plan=None,
                                   out=None, return_lse: bool = False):
    """Packed q [Tq, HQ, D] over paged caches, 16-bit or e4m3 with scales (see varlen_cache.py)."""
    q = _rows16(q)
    cu, seq, bt = _i32(cu_seqlens_q), _i32(cache_seqlens), _i32(block_table)
    Tq, HQ, D = q.shape
    if out is None:
        out = q.new_empty((Tq, HQ, D))
    lse = q.new_empty((Tq, HQ), dtype=torch.float32) if return_lse else None
    pages, PS, HKV, _ = k_cache.shape
    B = seq.shape[0]
    lib = _L()
    with _on(q):
        stream = _stream(q)
        if max_seqlen_q <= 1 and Tq and 0 < B <= _MAX_STEP_BATCH and (k_scales is None or (D == 128 and PS % 16 == 0)):
            # a decode step: the split-KV kernel reads K/V once for the query heads of a KV head
            # without a 128-row tile to fill
            q = _contig(q)
            splits, chunk = kvcache_plan(B, 1, HQ, HKV, D, max_seqlen_k)
            ws, ws_bytes = None, 0
            if splits > 1:
                ws_bytes = int(lib.mxfa_split_workspace_bytes(Tq * HQ, D, splits))
                ws = _scratch(q, stream, ws_bytes)
            counters = split_counters(q.device, stream, int(lib.mxfa_split_counter_bytes(B, 1, HQ, HKV)))
            name = "mxfa_kvcache_step_attention_launch"
            rc = lib.mxfa_kvcache_step_attention_launch(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scales), _lib.ptr(v_scales),
                cu.data_ptr(), seq.data_ptr(), bt.data_ptr(), None if plan is None else _lib.ptr(plan.order),
                out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, counters.data_ptr(), Tq, B, 1, HQ, HKV, D, PS,
                bt.shape[1], pages, splits, chunk, int(causal), _bf16(q), float(softmax_scale), stream)
            _lib.check(rc, name)
            return (out, lse) if return_lse else out
        table = ws = counters = None
        ws_bytes = 0
        if Tq and B and PS % 8 == 0 and HQ // HKV <= _MAX_GROUP:
            table = kvcache_chunk_plan(cu, seq, Tq, HQ, HKV, causal) if plan is None else plan.table
            ws_bytes, counter_bytes = _chunk_sizes(HKV, D)
            ws = _scratch(q, stream, ws_bytes)
            counters = split_counters(q.device, stream, counter_bytes)
            if k_scales is not None and unpack_pays(Tq, B, HQ // HKV, HKV, D, max_seqlen_k):
                rows = -(-max_seqlen_k // 128) * 128
                kv = q.new_empty((2, B, rows, HKV, D))
                pages_of = q.new_empty((B, 1), dtype=torch.int32)
                if q.dtype == torch.float16:
                    # fp16 does not hold every code * scale: tiles with such a value run on the cache itself
                    inexact = q.new_empty((int(lib.mxfa_unpack_flag_bytes(B, rows)) // 4,), dtype=torch.int32)
                    rc = lib.mxfa_kvcache_varlen_attention_half_launch(
                        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                        cu.data_ptr(), seq.data_ptr(), bt.data_ptr(), table.data_ptr(), table.numel() * 4,
                        out.data_ptr(), _lib.ptr(lse), ws.data_ptr(), ws_bytes, counters.data_ptr(), kv.data_ptr(),
                        kv[1].data_ptr(), pages_of.data_ptr(), inexact.data_ptr(), Tq, B, HQ, HKV, D, PS, bt.shape[1],
                        pages, rows, q.stride(0), q.stride(1), int(causal), float(softmax_scale), stream)
                    _lib.check(rc, "mxfa_kvcache_varlen_attention_half_launch")
                    return (out, lse) if return_lse else out
                rc = lib.mxfa_kvcache_unpack_launch(
                    k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), seq.data_ptr(),
                    bt.data_ptr(), kv.data_ptr(), kv[1].data_ptr(), pages_of.data_ptr(), B, rows, HKV, D, PS,
                    bt.shape[1], pages, _bf16(q), stream)
                _lib.check(rc, "mxfa_kvcache_unpack_launch")
                k_cache, v_cache, k_scales, v_scales, bt, pages, PS = kv[0], kv[1], None, None, pages_of, B, rows
        rc = lib.mxfa_kvcache_varlen_attention_launch(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scales), _lib.ptr(v_scales),
            cu.data_ptr(), seq.data_ptr(), bt.data_ptr(), _lib.ptr(table), 0 if table is None else table.numel() * 4,
            out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, _lib.ptr(counters), Tq, B, HQ, HKV, D,
            PS, bt.shape[1], pages, q.stride(0), q.stride(1), int(causal), _bf16(q), float(softmax_scale), stream)
    _lib.check(rc, "mxfa_kvcache_varlen_attention_launch")
    return (out, lse) if return_lse else out


# ------------------------------------------------------ combine / merge

def split_combine(ows, mdws, rows: int, head_dim: int, num_splits: int, dtype, *, lse: bool = False,
                  out=None):
    """LSE-merge split partials ows [rows, NP, D], mdws [rows, NP, 2] -> out [rows, D]."""
    if out is None:
        out = torch.empty((rows, head_dim), device=ows.device, dtype=dtype)
    lse_t = torch.empty((rows,), device=ows.device, dtype=torch.float32) if lse else None
    with _on(ows):
        rc = _L().mxfa_split_combine_launch(
            ows.data_ptr(), mdws.data_ptr(), out.data_ptr(), None, _lib.ptr(lse_t), rows, head_dim, num_splits,
            int(dtype == torch.bfloat16), _stream(ows))
    _lib.check(rc, "mxfa_split_combine_launch")
    return (out, lse_t) if lse else out


def lse_merge(packed, rows: int, head_dim: int, dtype, *, lse: bool = False, out=None):
    """Merge per-rank (O, LSE): packed f32 [N, rows, D + 1] -> out [rows, D] (and LSE)."""
    n_ranks = packed.shape[0]
    if out is None:
        out = torch.empty((rows, head_dim), device=packed.device, dtype=dtype)
    lse_t = torch.empty((rows,), device=packed.device, dtype=torch.float32) if lse else None
    with _on(packed):
        rc = _L().mxfa_lse_merge_launch(
            packed.data_ptr(), out.data_ptr(), _lib.ptr(lse_t), n_ranks, rows, head_dim,
            int(dtype == torch.bfloat16), _stream(packed))
    _lib.check(rc, "mxfa_lse_merge_launch")
    return (out, lse_t) if lse else out
