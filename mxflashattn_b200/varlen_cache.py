"""A ragged batch over a paged KV cache: write, read back, attend.

No reference counterpart (the reference appends and attends uniform blocks,
mxflashattn/reference.py:88-139); these are extensions of this package, used
next to ``flash_attn_with_kvcache`` by a serving loop that feeds prompts in
pieces, mixes pieces with decodes, or keeps its cache in 8 bits.

The batch is packed along the token axis: sequence ``b`` owns rows
``cu_seqlens[b]`` to ``cu_seqlens[b + 1]``, and they are the last of the
``cache_seqlens[b]`` tokens that its cache holds once the call's tokens are
in it (packed row ``t`` is position ``cache_seqlens[b] - cu_seqlens[b + 1] +
t``).  The same two vectors and the block table serve every call of a step
and every layer; no call changes them.

A quantised cache is a pair of ``torch.float8_e4m3fn`` tensors [P, PS, HKV, D]
with a pair of ``torch.float8_e8m0fnu`` scale tensors [P, HKV, PS]: one
power-of-two scale per token and KV head, value = code * scale.  Scales of one
sequence may lie as far apart as they like for K, within 2^100 of one another
for V; values under 2^-75 count as zero.

Calls validate on the host without reading device memory;
``MXFLASHATTN_STRICT_VALIDATION=1`` adds checks of the lengths and the table
that copy them to the host.
"""

from __future__ import annotations

import os
from dataclasses import dataclass

import torch

from .api import _resolved_scale
from .dispatch import dispatch
from .validation import validate_softmax_scale

_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu
_HALF = (torch.float16, torch.bfloat16)
_INDEX = (torch.int32, torch.int64)


def _require(ok: bool, message: str, error=ValueError) -> None:
    if not ok:
        raise error(message)


def _quick(check) -> bool:
    """Whether ``check()`` holds; arguments that are not tensors make it False.

    The checks below name what is wrong, one at a time, which costs a call
    more than its kernel's launch.  So each entry point asks one combined
    question first and goes through them only when its answer is no.
    """
    try:
        return check()
    except (AttributeError, TypeError, IndexError):
        return False


def _plain_caches(kc, vc, ks, vs) -> bool:
    s, d, dt = kc.shape, kc.device, kc.dtype
    if not (len(s) == 4 and vc.shape == s and vc.dtype == dt and vc.device == d and (s[3] == 128 or s[3] == 64)
            and s[0] > 0 and s[1] > 0 and s[2] > 0 and kc.is_contiguous() and vc.is_contiguous()):
        return False
    if dt != _E4M3:
        return dt in _HALF and ks is None and vs is None
    want = (s[0], s[2], s[1])
    return (ks.dtype == _E8M0 and vs.dtype == _E8M0 and ks.shape == want and vs.shape == want and ks.device == d
            and vs.device == d and ks.is_contiguous() and vs.is_contiguous())


def _plain_batch(cu, seq, bt, d) -> bool:
    b, w = bt.shape
    return (bt.dtype in _INDEX and cu.dtype in _INDEX and seq.dtype in _INDEX and seq.ndim == 1 and cu.ndim == 1
            and seq.shape[0] == b and cu.shape[0] == b + 1 and (w > 0 or b == 0) and cu.device == d
            and seq.device == d and bt.device == d)


def _validate_caches(k_cache, v_cache, k_scales, v_scales) -> bool:
    """Checks of a paged cache pair; True when it is quantised."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor", TypeError)
        _require(t.ndim == 4, f"{name} must have rank 4 with layout [pages, page_size, kv_heads, dim]")
    _require(k_cache.shape == v_cache.shape, "k_cache and v_cache must have identical shapes")
    _require(k_cache.dtype == v_cache.dtype, "k_cache and v_cache must have the same dtype")
    _require(k_cache.device == v_cache.device, "k_cache and v_cache must be on the same device")
    pages, page_size, kv_heads, dim = k_cache.shape
    _require(pages > 0 and page_size > 0 and kv_heads > 0, "the cache must have pages, page slots and kv heads")
    _require(dim in (64, 128), "head dimension must be 64 or 128")
    _require(k_cache.is_contiguous() and v_cache.is_contiguous(), "k_cache and v_cache must be contiguous")
    _require((k_scales is None) == (v_scales is None), "k_scales and v_scales must either both be provided or omitted")
    if k_cache.dtype != _E4M3:
        _require(k_cache.dtype in _HALF, "the cache must be float16, bfloat16 or float8_e4m3fn", TypeError)
        _require(k_scales is None, "k_scales / v_scales apply to float8_e4m3fn caches only")
        return False
    _require(k_scales is not None, "a float8_e4m3fn cache needs k_scales and v_scales")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor", TypeError)
        _require(t.dtype == _E8M0, f"{name} must be float8_e8m0fnu", TypeError)
        _require(t.shape == (pages, kv_heads, page_size) and t.is_contiguous() and t.device == k_cache.device,
                 f"{name} must be a contiguous [pages, kv_heads, page_size] tensor on the cache's device")
    return True


def _validate_batch(cu_seqlens, cache_seqlens, block_table, device, cu_name="cu_seqlens") -> int:
    """Checks of the ragged batch's index tensors; the batch size."""
    for name, t, ndim in ((cu_name, cu_seqlens, 1), ("cache_seqlens", cache_seqlens, 1),
                          ("block_table", block_table, 2)):
        if t is None and name == "block_table":
            continue
        _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor", TypeError)
        _require(t.ndim == ndim, f"{name} must have rank {ndim}")
        _require(t.dtype in (torch.int32, torch.int64), f"{name} must use int32 or int64", TypeError)
        _require(t.device == device, f"{name} must be on the same device as the cache")
    batch = cache_seqlens.numel()
    _require(cu_seqlens.numel() == batch + 1, f"{cu_name} must have one entry more than cache_seqlens")
    if block_table is not None:
        _require(block_table.shape[0] == batch, "block_table must have one row per sequence")
        _require(block_table.shape[1] > 0 or batch == 0, "block_table must have at least one column")
    return batch


def _strict_batch_checks(cu_seqlens, cache_seqlens, block_table, total, page_size, pages, must_fit) -> None:
    """Host-syncing checks of MXFLASHATTN_STRICT_VALIDATION=1."""
    offsets = [int(x) for x in cu_seqlens.detach().cpu().tolist()]
    lengths = [int(x) for x in cache_seqlens.detach().cpu().tolist()]
    if offsets[0] != 0 or any(b < a for a, b in zip(offsets, offsets[1:])) or offsets[-1] > total:
        raise ValueError("cu_seqlens must start at zero, not decrease, and stay within the packed tokens")
    if any(n < 0 for n in lengths):
        raise ValueError("cache sequence lengths must be non-negative")
    if must_fit and any(b - a > n for a, b, n in zip(offsets, offsets[1:], lengths)):
        raise ValueError("cache_seqlens must count the call's own tokens")
    if block_table is None:
        return
    for n, row in zip(lengths, block_table.detach().cpu().tolist()):
        used = (n + page_size - 1) // page_size
        if used > len(row):
            raise ValueError("block_table does not contain enough pages for cache sequence")
        if any(int(pg) < 0 or int(pg) >= pages for pg in row[:used]):
            raise ValueError("block_table contains an out-of-range page index")


def _strict() -> bool:
    return os.getenv("MXFLASHATTN_STRICT_VALIDATION", "0") == "1"


def _validate_append(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, k_scales, v_scales) -> None:
    quant = _validate_caches(k_cache, v_cache, k_scales, v_scales)
    for name, t in (("k", k), ("v", v)):
        _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor", TypeError)
        _require(t.ndim == 3 and t.shape[1:] == k_cache.shape[2:],
                 f"{name} must have rank 3 with layout [total_tokens, kv_heads, dim] matching the cache")
        _require(t.device == k_cache.device, f"{name} must be on the cache's device")
        _require(t.dtype in _HALF, f"{name} must be float16 or bfloat16", TypeError)
    _require(k.shape == v.shape, "k and v must have identical shapes")
    _require(k.dtype == v.dtype, "k and v must have the same dtype")
    _require(quant or k.dtype == k_cache.dtype, "k and v must have the cache's dtype")
    _validate_batch(cu_seqlens, cache_seqlens, block_table, k_cache.device)
    _require(block_table is not None, "block_table is required")


def kvcache_append_varlen(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cu_seqlens: torch.Tensor,
    cache_seqlens: torch.Tensor,
    block_table: torch.Tensor,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
) -> None:
    """Write packed ``k``/``v`` [T, HKV, D] into a paged cache, in place.

    ``cache_seqlens`` counts the new tokens (see the module's text).  A 16-bit
    cache of ``k``'s dtype receives a bit-exact copy.  A quantised cache
    receives e4m3 codes of ``x / s`` and the scales: ``s`` is the smallest
    power of two (at least 2^-126) with ``max |x| <= 448 s`` over the row's
    finite values; an infinity saturates to ``448 s`` and a NaN stays NaN.
    ``k`` and ``v`` may be strided views (slices of a fused projection); rows
    before ``cu_seqlens[0]`` or past ``cu_seqlens[-1]`` belong to no sequence and
    are not written.
    """
    if not _quick(lambda: _plain_caches(k_cache, v_cache, k_scales, v_scales)
                  and _plain_batch(cu_seqlens, cache_seqlens, block_table, k_cache.device)
                  and k.ndim == 3 and k.shape == v.shape and k.shape[1:] == k_cache.shape[2:] and k.dtype == v.dtype
                  and k.dtype in _HALF and (k_scales is not None or k.dtype == k_cache.dtype)
                  and k.device == k_cache.device and v.device == k_cache.device):
        _validate_append(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, k_scales, v_scales)
    if _strict():
        _strict_batch_checks(cu_seqlens, cache_seqlens, block_table, k.shape[0], k_cache.shape[1], k_cache.shape[0],
                             True)
    dispatch("kvcache_append_varlen", k,
             (k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, k_scales, v_scales))


def kvcache_gather_varlen(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cu_seqlens: torch.Tensor,
    cache_seqlens: torch.Tensor,
    block_table: torch.Tensor,
    total_tokens: int,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Read the last ``cu_seqlens[b + 1] - cu_seqlens[b]`` tokens of every sequence back, packed.

    Returns ``(k, v)`` [total_tokens, HKV, D]: the cache's values, for a
    quantised cache ``code * scale`` rounded once to ``dtype`` (float16 or
    bfloat16, the default).  A 16-bit cache is copied bit for bit.  Rows that
    no sequence owns, or whose page the table does not have, are zero.
    """
    quant = k_scales is not None
    if not _quick(lambda: _plain_caches(k_cache, v_cache, k_scales, v_scales)
                  and _plain_batch(cu_seqlens, cache_seqlens, block_table, k_cache.device)):
        quant = _validate_caches(k_cache, v_cache, k_scales, v_scales)
        _validate_batch(cu_seqlens, cache_seqlens, block_table, k_cache.device)
        _require(block_table is not None, "block_table is required")
    if dtype is None:
        dtype = torch.bfloat16 if quant else k_cache.dtype
    if not (dtype in _HALF and (quant or dtype == k_cache.dtype)):
        _require(dtype in _HALF, "dtype must be float16 or bfloat16", TypeError)
        _require(quant or dtype == k_cache.dtype, "a 16-bit cache is read back in its own dtype")
    total_tokens = int(total_tokens)
    if total_tokens < 0:
        raise ValueError("total_tokens must be non-negative")
    if _strict():
        _strict_batch_checks(cu_seqlens, cache_seqlens, block_table, total_tokens, k_cache.shape[1],
                             k_cache.shape[0], True)
    shape = (total_tokens, *k_cache.shape[2:])
    k = k_cache.new_empty(shape, dtype=dtype)
    v = k_cache.new_empty(shape, dtype=dtype)
    dispatch("kvcache_gather_varlen", k,
             (k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, k_scales, v_scales, k, v))
    return k, v


@dataclass(frozen=True)
class KvChunkPlan:
    """How one step's ragged batch is divided (``kvcache_chunk_plan``); every layer of the step uses it.

    On the device: ``table``, the items of the tiled kernel, and for a decode
    step ``order``, the sequences longest first.
    """

    total_q: int
    batch: int
    max_seqlen_q: int
    q_heads: int
    kv_heads: int
    causal: bool
    table: torch.Tensor | None
    order: torch.Tensor | None = None
    device: torch.device | None = None


def kvcache_chunk_plan(
    cu_seqlens_q: torch.Tensor,
    cache_seqlens: torch.Tensor,
    total_q: int,
    max_seqlen_q: int,
    *,
    q_heads: int,
    kv_heads: int,
    causal: bool = False,
) -> KvChunkPlan:
    """The division of a step's ragged batch for ``flash_attn_varlen_with_kvcache(..., plan=)``.

    One small kernel reads the lengths and writes the plan on the device.
    Call it once per step, after the lengths are final, and pass the result
    to every layer of that step; a call without a plan makes its own.  A plan
    belongs to the lengths it was made from: after they change, make another.
    """
    for name, t in (("cu_seqlens_q", cu_seqlens_q), ("cache_seqlens", cache_seqlens)):
        _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor", TypeError)
    _require(cu_seqlens_q.device.type == "cuda", "cu_seqlens_q must be on a CUDA device")
    batch = _validate_batch(cu_seqlens_q, cache_seqlens, None, cu_seqlens_q.device, "cu_seqlens_q")
    _require(int(total_q) >= 0 and int(max_seqlen_q) >= 0, "total_q and max_seqlen_q must be non-negative")
    _require(q_heads > 0 and kv_heads > 0 and q_heads % kv_heads == 0,
             "q heads must be a positive multiple of kv heads")
    from . import backend

    table = backend.kvcache_chunk_plan(cu_seqlens_q, cache_seqlens, int(total_q), q_heads, kv_heads, causal)
    return KvChunkPlan(int(total_q), batch, int(max_seqlen_q), int(q_heads), int(kv_heads), bool(causal), table,
                       backend.kvcache_length_order(cache_seqlens) if max_seqlen_q <= 1 and batch else None,
                       cu_seqlens_q.device)


def _plan_fits(plan, q, k_cache, cache_seqlens, max_seqlen_q, causal) -> bool:
    """Whether ``plan`` was made for a batch of these counts."""
    return (plan.total_q == q.shape[0] and plan.batch == cache_seqlens.shape[0] and plan.max_seqlen_q == max_seqlen_q
            and plan.q_heads == q.shape[1] and plan.kv_heads == k_cache.shape[2] and plan.causal == bool(causal)
            and plan.device == q.device)


def _validate_attention(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, max_seqlen_q, max_seqlen_k,
                        softmax_scale, causal, k_scales, v_scales, plan, out) -> None:
    validate_softmax_scale(softmax_scale)
    quant = _validate_caches(k_cache, v_cache, k_scales, v_scales)
    _require(isinstance(q, torch.Tensor), "q must be a torch.Tensor", TypeError)
    _require(q.ndim == 3, "q must have rank 3 with layout [total_tokens, heads, dim]")
    _require(q.device == k_cache.device, "q must be on the cache's device")
    _require(q.shape[2] == k_cache.shape[3], "q and the cache must have the same head dimension")
    _require(q.shape[1] > 0 and q.shape[1] % k_cache.shape[2] == 0, "q heads must be a positive multiple of kv heads")
    _require(q.dtype in _HALF, "q must be float16 or bfloat16", TypeError)
    _require(quant or q.dtype == k_cache.dtype, "q must have the cache's dtype")
    _validate_batch(cu_seqlens_q, cache_seqlens, block_table, k_cache.device, "cu_seqlens_q")
    _require(block_table is not None, "block_table is required")
    _require(max_seqlen_q >= 0, "max_seqlen_q must be non-negative")
    _require(max_seqlen_k is None or max_seqlen_k >= 0, "max_seqlen_k must be non-negative")
    if plan is not None:
        _require(isinstance(plan, KvChunkPlan), "plan must come from kvcache_chunk_plan", TypeError)
        _require(_plan_fits(plan, q, k_cache, cache_seqlens, max_seqlen_q, causal),
                 "plan was made for another batch")
    if out is not None:
        _require(isinstance(out, torch.Tensor) and out.shape == q.shape and out.dtype == q.dtype
                 and out.device == q.device and out.is_contiguous(),
                 "out must be a contiguous tensor with q's shape, dtype and device")


def flash_attn_varlen_with_kvcache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cache_seqlens: torch.Tensor,
    block_table: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int | None = None,
    *,
    softmax_scale: float | None = None,
    causal: bool = False,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    plan: KvChunkPlan | None = None,
    out: torch.Tensor | None = None,
    return_softmax_lse: bool = False,
):
    """Attention of packed queries [Tq, HQ, D] over each sequence's cached tokens.

    The queries' own K and V are in the cache already
    (``kvcache_append_varlen``), so ``cache_seqlens`` counts them; with
    ``causal`` the query at position ``p`` sees keys ``0 .. p``.  Pieces of
    prompts and single decode tokens may be mixed.  ``max_seqlen_q`` bounds
    the queries of one sequence, ``max_seqlen_k`` (default: what the table
    can hold) the cached tokens: no sequence may be longer (a longer one may be
    cut and flagged).  A row that sees no key is 0 with LSE -inf;
    rows before ``cu_seqlens_q[0]`` or past ``cu_seqlens_q[-1]`` are padding and
    are not written.

    The cache is 16-bit in ``q``'s dtype, or quantised with ``k_scales`` and
    ``v_scales``.  ``plan`` comes from ``kvcache_chunk_plan`` for the same
    lengths.  ``out`` (contiguous, ``q``'s shape, dtype and device) receives
    the result.  With ``return_softmax_lse`` the natural-log LSE [Tq, HQ]
    (float32) is returned too.
    """
    max_seqlen_q = int(max_seqlen_q)
    max_seqlen_k = None if max_seqlen_k is None else int(max_seqlen_k)
    if softmax_scale is not None or not _quick(
            lambda: _plain_caches(k_cache, v_cache, k_scales, v_scales)
            and _plain_batch(cu_seqlens_q, cache_seqlens, block_table, k_cache.device)
            and q.ndim == 3 and q.shape[2] == k_cache.shape[3] and q.shape[1] > 0
            and q.shape[1] % k_cache.shape[2] == 0 and q.device == k_cache.device
            and q.dtype in _HALF and (k_scales is not None or q.dtype == k_cache.dtype)
            and max_seqlen_q >= 0 and (max_seqlen_k is None or max_seqlen_k >= 0)
            and (plan is None or _plan_fits(plan, q, k_cache, cache_seqlens, max_seqlen_q, causal))
            and (out is None or (out.shape == q.shape and out.dtype == q.dtype and out.device == q.device
                                 and out.is_contiguous()))):
        _validate_attention(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, max_seqlen_q, max_seqlen_k,
                            softmax_scale, causal, k_scales, v_scales, plan, out)
    capacity = block_table.shape[1] * k_cache.shape[1]
    if max_seqlen_k is None or max_seqlen_k > capacity:
        max_seqlen_k = capacity
    if _strict():
        _strict_batch_checks(cu_seqlens_q, cache_seqlens, block_table, q.shape[0], k_cache.shape[1],
                             k_cache.shape[0], False)
    return dispatch("flash_attn_varlen_with_kvcache", q,
                    (q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, max_seqlen_q,
                     max_seqlen_k, _resolved_scale(q.shape[-1], softmax_scale), bool(causal), k_scales,
                     v_scales, plan, out, bool(return_softmax_lse)))
