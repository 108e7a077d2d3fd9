"""FlashInfer-shaped page-table and append functions, backed by libpagedkv.so.

Same names, argument order, keywords and result shapes as the FlashInfer 0.6.5 calls the
reference makes (ecahlang/manager.py:143-146, 155-165, 170-185, 271-280), so the manager and
any FlashInfer caller can switch by changing the import.
"""
from __future__ import annotations

from typing import Tuple, Union

import torch

from ._lib import (CALL_APPEND_FP8, CALL_NORM_ROPE, CALL_READ_FP8, DTYPE_CODE, call, check, dtype_code, lib,
                   stream_ptr)

CacheT = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _i32(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_cuda:
        raise ValueError(f"{name} must be an int32 CUDA tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


class CacheView:
    """K/V base pointers and geometry of one layer's paged cache.

    Accepts the single-tensor NHD form ``[pages, 2, page_size, Hkv, D]`` the reference
    allocates (ecahlang/manager.py:51-54, indexed per layer at :160) or a ``(k_cache,
    v_cache)`` pair of ``[pages, page_size, Hkv, D]`` tensors.
    """

    __slots__ = ("k_ptr", "v_ptr", "page_stride", "num_pages", "page_size", "num_kv_heads",
                 "head_dim", "dtype", "device")

    def __init__(self, paged_kv_cache: CacheT, kv_layout: str = "NHD"):
        (self.k_ptr, self.v_ptr, self.page_stride, self.num_pages, self.page_size, self.num_kv_heads, self.head_dim,
         self.dtype, self.device) = cache_fields(paged_kv_cache, kv_layout)


def cache_fields(paged_kv_cache: CacheT, kv_layout: str = "NHD") -> tuple:
    """A ``CacheView``'s fields in order, for calls where the object's own time counts."""
    if kv_layout != "NHD" and kv_layout.upper() != "NHD":
        raise NotImplementedError("only the NHD cache layout is implemented (the reference uses NHD)")
    if isinstance(paged_kv_cache, (tuple, list)):
        k, v = paged_kv_cache
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("(k_cache, v_cache) must both be [pages, page_size, Hkv, D]")
        for t in (k, v):
            if not t.is_contiguous():
                raise ValueError("k_cache / v_cache must be contiguous")
        pages, ps, hkv, d = k.shape
        kp, vp, stride = k.data_ptr(), v.data_ptr(), k.stride(0)
    else:
        k = paged_kv_cache
        shape = k.shape
        if len(shape) != 5 or shape[1] != 2:
            raise ValueError("paged_kv_cache must be [pages, 2, page_size, Hkv, D] (NHD)")
        if not k.is_contiguous():
            raise ValueError("paged_kv_cache must be contiguous")
        pages, _, ps, hkv, d = shape
        kp = k.data_ptr()
        half = ps * hkv * d
        vp = kp + half * k.element_size() if kp else 0
        stride = 2 * half
    if not k.is_cuda:
        raise ValueError("paged_kv_cache must live on a CUDA (HIP) device")
    return kp, vp, stride, pages, ps, hkv, d, k.dtype, k.device


FP8 = torch.float8_e4m3fn


def scale_fields(kv_scales, pages: int, ps: int, hkv: int, dtype: torch.dtype, dev: torch.device) -> tuple:
    """(K address, V address, bytes between pages) of the scales (``new_kv_scales``) of a cache of these sizes."""
    if dtype is not FP8:
        raise ValueError(f"kv_scales go with a float8_e4m3fn cache, not {dtype}")
    if kv_scales is None:
        raise ValueError("a float8_e4m3fn cache needs kv_scales")
    if isinstance(kv_scales, (tuple, list)):
        if len(kv_scales) != 2:
            raise ValueError("kv_scales must be one tensor or a (k_scales, v_scales) pair")
        for t in kv_scales:
            _check_scales(t, (pages, hkv, ps), dev)
        return kv_scales[0].data_ptr(), kv_scales[1].data_ptr(), hkv * ps
    _check_scales(kv_scales, (pages, 2, hkv, ps), dev)
    p, n = kv_scales.data_ptr(), hkv * ps
    return p, p + n if p else 0, 2 * n


def _check_scales(t, want: tuple, dev: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float8_e8m0fnu or t.shape != want:
        raise ValueError(f"kv_scales must be float8_e8m0fnu {list(want)}")
    if not t.is_contiguous():
        raise ValueError("kv_scales must be contiguous")
    if t.device != dev:
        raise ValueError(f"kv_scales are on {t.device}, the cache on {dev}")


def new_kv_scales(paged_kv_cache: torch.Tensor) -> torch.Tensor:
    """Scales for an 8-bit cache (``torch.float8_e4m3fn``, same shapes as the others): one power of two a token and
    KV head, ``torch.float8_e8m0fnu`` of shape ``[..., pages, 2, Hkv, page_size]`` for a cache ``[..., pages, 2,
    page_size, Hkv, D]``, here of ones.  A stored value is code * scale.  With a ``(k_cache, v_cache)`` pair goes a
    ``(k_scales, v_scales)`` pair of ``[pages, Hkv, page_size]``."""
    *lead, two, ps, hkv, _ = paged_kv_cache.shape
    if two != 2 or paged_kv_cache.dtype != FP8:
        raise ValueError("paged_kv_cache must be float8_e4m3fn [..., pages, 2, page_size, Hkv, D]")
    return torch.full((*lead, 2, hkv, ps), 127, dtype=torch.uint8, device=paged_kv_cache.device).view(torch.float8_e8m0fnu)


def get_seq_lens(kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor, page_size: int) -> torch.Tensor:
    """seq_len[b] = max(indptr[b+1]-indptr[b]-1, 0) * page_size + last_page_len[b] (int32)."""
    _i32(kv_indptr, "kv_indptr")
    _i32(kv_last_page_len, "kv_last_page_len")
    b = kv_last_page_len.numel()
    if kv_indptr.numel() != b + 1:
        raise ValueError("kv_indptr must have batch+1 entries")
    out = torch.empty(b, dtype=torch.int32, device=kv_indptr.device)
    check(lib().pkv_get_seq_lens(kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), b,
                                 int(page_size), out.data_ptr(), stream_ptr(kv_indptr.device)),
          "get_seq_lens")
    return out


def get_batch_indices_positions(append_indptr: torch.Tensor, seq_lens: torch.Tensor, nnz) -> tuple:
    """(batch_indices, positions) of the nnz appended tokens, both int32 [nnz].

    ``nnz`` may be an int or a 0-d tensor (the reference passes ``append_indptr[-1]``,
    ecahlang/manager.py:145); a device tensor costs one host sync, as in the reference.
    """
    _i32(append_indptr, "append_indptr")
    _i32(seq_lens, "seq_lens")
    nnz = int(nnz)
    b = seq_lens.numel()
    if append_indptr.numel() != b + 1:
        raise ValueError("append_indptr must have batch+1 entries")
    dev = append_indptr.device
    bidx = torch.empty(nnz, dtype=torch.int32, device=dev)
    pos = torch.empty(nnz, dtype=torch.int32, device=dev)
    if nnz:
        check(lib().pkv_get_batch_indices_positions(append_indptr.data_ptr(), seq_lens.data_ptr(), b,
                                                    nnz, bidx.data_ptr(), pos.data_ptr(),
                                                    stream_ptr(dev)),
              "get_batch_indices_positions")
    return bidx, pos


def _row_strides(t: torch.Tensor, name: str) -> tuple:
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name} must be [nnz, heads, head_dim] with a unit inner stride")
    return t.stride(0), t.stride(1)


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor,
                          batch_indices: torch.Tensor, positions: torch.Tensor,
                          paged_kv_cache: CacheT, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                          kv_last_page_len: torch.Tensor, kv_layout: str = "NHD",
                          err_count: torch.Tensor | None = None, kv_scales=None) -> None:
    """Scatter ``append_key/value[i]`` into page ``kv_indices[kv_indptr[b] + pos // ps]`` slot
    ``pos % ps`` with b = batch_indices[i], pos = positions[i].  Bit-exact copy.

    ``kv_last_page_len`` is accepted for signature parity and, as in the reference's
    dependency, not used by the scatter.  ``err_count`` (optional int32 [1]) counts tokens
    whose metadata falls outside their sequence's pages; they are skipped.

    With an 8-bit cache (``torch.float8_e4m3fn``) and its ``kv_scales`` (see ``new_kv_scales``) the rows, fp16,
    bf16 or fp32, are quantised as they are written: each (token, head) row gets the smallest power of
    two s >= 2^-126 with max|x| <= 448 s as its scale and is stored as the e4m3 values nearest to x / s.
    Elements that are not finite are stored as NaN.  head_dim must be a multiple of 16, up to 512.  Of two
    tokens in one slot either's codes may meet the other's scale.
    """
    if kv_scales is not None:
        return _append_fp8(append_key, append_value, paged_kv_cache, kv_layout, kv_scales, err_count, batch_indices, positions,
                           kv_indices, kv_indptr)
    cv = CacheView(paged_kv_cache, kv_layout)
    if cv.dtype is FP8:
        raise ValueError("a float8_e4m3fn cache needs kv_scales")
    for t, n in ((append_key, "append_key"), (append_value, "append_value")):
        if t.dtype != cv.dtype:
            raise ValueError(f"{n} dtype {t.dtype} differs from the cache dtype {cv.dtype}")
        if t.shape[1:] != (cv.num_kv_heads, cv.head_dim):
            raise ValueError(f"{n} must be [nnz, {cv.num_kv_heads}, {cv.head_dim}]")
    nnz = append_key.shape[0]
    if append_value.shape[0] != nnz or batch_indices.numel() < nnz or positions.numel() < nnz:
        raise ValueError("append_key, append_value, batch_indices and positions disagree on nnz")
    _i32(batch_indices, "batch_indices")
    _i32(positions, "positions")
    _i32(kv_indices, "kv_indices")
    _i32(kv_indptr, "kv_indptr")
    ksn, ksh = _row_strides(append_key, "append_key")
    vsn, vsh = _row_strides(append_value, "append_value")
    err_ptr = 0
    if err_count is not None:
        err_ptr = _i32(err_count, "err_count").data_ptr()
    if nnz == 0:
        return
    check(lib().pkv_append_paged_kv_cache(
        append_key.data_ptr(), ksn, ksh, append_value.data_ptr(), vsn, vsh,
        batch_indices.data_ptr(), positions.data_ptr(), nnz, cv.k_ptr, cv.v_ptr, cv.page_stride,
        cv.num_pages, kv_indices.data_ptr(), kv_indices.numel(), kv_indptr.data_ptr(),
        kv_indptr.numel() - 1,
        cv.num_kv_heads, cv.head_dim, cv.page_size, dtype_code(cv.dtype), err_ptr,
        stream_ptr(cv.device)), "append_paged_kv_cache")


def _ids(t: torch.Tensor, name: str, dev: torch.device) -> int:
    """Address of an int32 index tensor on the cache's device."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or not t.is_contiguous():
        _i32(t, name)
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the cache on {dev}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, shape: tuple, dt: torch.dtype, dev: torch.device) -> tuple:
    """Strides of [n, heads, head_dim] rows, whose type, shape and place are checked."""
    st = t.stride()
    if t.dtype is not dt or t.shape != shape or st[2] != 1:
        raise ValueError(f"{name} must be {list(shape)} in {dt} with a unit inner stride")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the cache on {dev}")
    return st


_ROW_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _row_dtype(t: torch.Tensor, d: int) -> torch.dtype:
    dt = t.dtype
    if dt not in _ROW_DTYPES:
        raise ValueError(f"rows must be float16, bfloat16 or float32, not {dt}")
    if d % 16 or not 0 < d <= 512:
        raise ValueError("head_dim must be a multiple of 16, up to 512")
    return dt


def _append_fp8(append_key, append_value, paged_kv_cache, kv_layout, kv_scales, err_count, batch_indices=None, positions=None,
                kv_indices=None, kv_indptr=None, slots=None) -> None:
    """The append into an 8-bit cache, by page table or slots."""
    kp, vp, page_stride, pages, ps, hkv, d, cdt, dev = cache_fields(paged_kv_cache, kv_layout)
    scales = scale_fields(kv_scales, pages, ps, hkv, cdt, dev)
    dt = _row_dtype(append_key, d)
    nnz = append_key.shape[0]
    shape = (nnz, hkv, d)
    ks, vs = _rows(append_key, "append_key", shape, dt, dev), _rows(append_value, "append_value", shape, dt, dev)
    bi = po = sl = idx = nidx = ptr = batch = err = 0
    if slots is not None:
        sl = _ids(slots, "slots", dev)
        if slots.numel() < nnz:
            raise ValueError("append_key, append_value and slots disagree on nnz")
    else:
        bi, po = _ids(batch_indices, "batch_indices", dev), _ids(positions, "positions", dev)
        if batch_indices.numel() < nnz or positions.numel() < nnz:
            raise ValueError("append_key, append_value, batch_indices and positions disagree on nnz")
        idx, nidx = _ids(kv_indices, "kv_indices", dev), kv_indices.numel()
        ptr, batch = _ids(kv_indptr, "kv_indptr", dev), kv_indptr.numel() - 1
        if batch < 0:
            raise ValueError("kv_indptr must have batch+1 entries")
    if err_count is not None:
        err = _ids(err_count, "err_count", dev)
    if nnz == 0:
        return
    check(call(CALL_APPEND_FP8, append_key.data_ptr(), ks[0], ks[1], append_value.data_ptr(), vs[0], vs[1], bi, po, sl, nnz,
               kp, vp, page_stride, pages, *scales, idx, nidx, ptr, batch, hkv, d, ps, DTYPE_CODE[dt], err, stream_ptr(dev)),
          "append_paged_kv_cache (8-bit cache)")


def append_paged_kv_cache_slots(append_key: torch.Tensor, append_value: torch.Tensor, slots: torch.Tensor,
                                paged_kv_cache: CacheT, kv_layout: str = "NHD",
                                err_count: torch.Tensor | None = None, kv_scales=None) -> None:
    """``append_paged_kv_cache`` with each token's destination resolved beforehand: token i goes
    to page ``slots[i] // ps``, slot ``slots[i] % ps`` (``slots`` as the page-table gather of
    ``AutoKVCacheManager.fill_cuda_graph_metadata`` writes them).  One lookup per token instead
    of the three dependent ones through batch_indices / positions, kv_indptr and kv_indices;
    the bytes written are the same.  Tokens with a negative or out-of-pool slot are skipped and
    counted in ``err_count``.  With an 8-bit cache and its ``kv_scales`` the rows are quantised as
    ``append_paged_kv_cache`` does it.
    """
    if kv_scales is not None:
        return _append_fp8(append_key, append_value, paged_kv_cache, kv_layout, kv_scales, err_count, slots=slots)
    cv = CacheView(paged_kv_cache, kv_layout)
    if cv.dtype is FP8:
        raise ValueError("a float8_e4m3fn cache needs kv_scales")
    for t, n in ((append_key, "append_key"), (append_value, "append_value")):
        if t.dtype != cv.dtype:
            raise ValueError(f"{n} dtype {t.dtype} differs from the cache dtype {cv.dtype}")
        if t.shape[1:] != (cv.num_kv_heads, cv.head_dim):
            raise ValueError(f"{n} must be [nnz, {cv.num_kv_heads}, {cv.head_dim}]")
    nnz = append_key.shape[0]
    if append_value.shape[0] != nnz or slots.numel() < nnz:
        raise ValueError("append_key, append_value and slots disagree on nnz")
    _i32(slots, "slots")
    ksn, ksh = _row_strides(append_key, "append_key")
    vsn, vsh = _row_strides(append_value, "append_value")
    err_ptr = 0
    if err_count is not None:
        err_ptr = _i32(err_count, "err_count").data_ptr()
    if nnz == 0:
        return
    check(lib().pkv_append_paged_kv_cache_slots(
        append_key.data_ptr(), ksn, ksh, append_value.data_ptr(), vsn, vsh, slots.data_ptr(), nnz,
        cv.k_ptr, cv.v_ptr, cv.page_stride, cv.num_pages, cv.num_kv_heads, cv.head_dim, cv.page_size,
        dtype_code(cv.dtype), err_ptr, stream_ptr(cv.device)), "append_paged_kv_cache_slots")


def append_paged_kv_cache_with_rope(q: torch.Tensor, append_key: torch.Tensor, append_value: torch.Tensor,
                                    cos: torch.Tensor, sin: torch.Tensor, batch_indices: torch.Tensor,
                                    positions: torch.Tensor, paged_kv_cache: CacheT,
                                    kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                                    kv_last_page_len: torch.Tensor, kv_layout: str = "NHD",
                                    q_out: torch.Tensor | None = None,
                                    err_count: torch.Tensor | None = None) -> torch.Tensor:
    """The model's rotary embedding on the new tokens, then the append, in one launch.

    Equivalent, bit for bit, to ``q, k = apply_rotary_pos_emb(q, k, cos, sin)`` as the model
    runs it (transformers/models/qwen2/modeling_qwen2.py:210-211) followed by
    ``append_paged_kv_cache(k, append_value, ...)`` (ecahlang/main.py:62-66).  ``q``,
    ``append_key`` and ``append_value`` are ``[nnz, heads, head_dim]`` row views; ``cos`` /
    ``sin`` are the tokens' ``[nnz, head_dim]`` position-embedding rows in the cache dtype.
    The rotated queries go to ``q_out`` (default: a new tensor; pass ``q`` to rotate in
    place) and are returned.  The rotated keys exist only in the cache.
    """
    cv = CacheView(paged_kv_cache, kv_layout)
    for t, n in ((append_key, "append_key"), (append_value, "append_value")):
        if t.dtype != cv.dtype:
            raise ValueError(f"{n} dtype {t.dtype} differs from the cache dtype {cv.dtype}")
        if t.shape[1:] != (cv.num_kv_heads, cv.head_dim):
            raise ValueError(f"{n} must be [nnz, {cv.num_kv_heads}, {cv.head_dim}]")
    nnz = append_key.shape[0]
    if q.dtype != cv.dtype or q.dim() != 3 or q.shape[0] != nnz or q.shape[2] != cv.head_dim:
        raise ValueError(f"q must be [{nnz}, Hq, {cv.head_dim}] in {cv.dtype}")
    for t, n in ((cos, "cos"), (sin, "sin")):
        if t.dtype != cv.dtype or t.dim() != 2 or t.shape != (nnz, cv.head_dim) or t.stride(1) != 1:
            raise ValueError(f"{n} must be [{nnz}, {cv.head_dim}] in {cv.dtype} with a unit inner stride")
    if cos.stride(0) != sin.stride(0):
        raise ValueError("cos and sin must share a row stride")
    if cv.head_dim % 8:
        raise ValueError("head_dim must be a multiple of 8")
    if append_value.shape[0] != nnz or batch_indices.numel() < nnz or positions.numel() < nnz:
        raise ValueError("q, append_key, append_value, batch_indices and positions disagree on nnz")
    if q_out is None:
        q_out = torch.empty_like(q)
    elif q_out.shape != q.shape or q_out.dtype != q.dtype:
        raise ValueError("q_out must match q's shape and dtype")
    _i32(batch_indices, "batch_indices")
    _i32(positions, "positions")
    _i32(kv_indices, "kv_indices")
    _i32(kv_indptr, "kv_indptr")
    qsn, qsh = _row_strides(q, "q")
    osn, osh = _row_strides(q_out, "q_out")
    ksn, ksh = _row_strides(append_key, "append_key")
    vsn, vsh = _row_strides(append_value, "append_value")
    for t, n in ((q, "q"), (q_out, "q_out"), (append_key, "append_key"), (append_value, "append_value"),
                 (cos, "cos"), (sin, "sin"), (batch_indices, "batch_indices"), (positions, "positions")):
        if t.device != cv.device:
            raise ValueError(f"{n} is on {t.device}, the cache on {cv.device}")
    err_ptr = 0
    if err_count is not None:
        err_ptr = _i32(err_count, "err_count").data_ptr()
    if nnz == 0:
        return q_out
    check(lib().pkv_append_paged_kv_cache_rope(
        q.data_ptr(), qsn, qsh, q_out.data_ptr(), osn, osh, q.shape[1],
        append_key.data_ptr(), ksn, ksh, append_value.data_ptr(), vsn, vsh,
        cos.data_ptr(), sin.data_ptr(), cos.stride(0),
        batch_indices.data_ptr(), positions.data_ptr(), nnz, cv.k_ptr, cv.v_ptr, cv.page_stride,
        cv.num_pages, kv_indices.data_ptr(), kv_indices.numel(), kv_indptr.data_ptr(),
        kv_indptr.numel() - 1, cv.num_kv_heads, cv.head_dim, cv.page_size, dtype_code(cv.dtype), err_ptr,
        stream_ptr(cv.device)), "append_paged_kv_cache_with_rope")
    return q_out


def append_paged_kv_cache_with_norm_rope(q: torch.Tensor, append_key: torch.Tensor, append_value: torch.Tensor,
                                         q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                                         cos: torch.Tensor, sin: torch.Tensor, batch_indices: torch.Tensor,
                                         positions: torch.Tensor, paged_kv_cache: CacheT,
                                         kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                                         kv_last_page_len: torch.Tensor, kv_layout: str = "NHD", eps: float = 1e-6,
                                         q_out: torch.Tensor | None = None, err_count: torch.Tensor | None = None,
                                         kv_scales=None) -> torch.Tensor:
    """RMS norm of every query and key head, rotary embedding and append, in one launch: what a model with
    per-head query / key norms does between its projections and the attention.

    ``y = x / sqrt(mean(x^2) + eps) * weight`` over the head_dim of each row of ``q`` and ``append_key``, then
    ``y * cos + rotate_half(y) * sin``, all in fp32 and rounded once: the queries into ``q_out`` (default: a new
    tensor; pass ``q`` to work in place), which is returned, the keys into their pages.  Values are appended
    unchanged.  ``q_weight`` / ``k_weight`` ``[head_dim]`` (``None``: rows of that kind are rotated only; both of
    one type) and ``cos`` / ``sin`` ``[nnz, head_dim]`` are in the rows' type or fp32; a weight that a model
    keeps as an offset from one is passed as ``1 + w``.  The cache is in the rows' type, or an 8-bit one with
    its ``kv_scales``: then keys and values are quantised as ``append_paged_kv_cache`` does it, the keys as if
    they had been computed exactly (where an fp32 key is next to a tie, it is computed again in 64 bits).
    head_dim must be a multiple of 16, up to 512.  Tokens with bad metadata are skipped, but for their
    queries, and counted in ``err_count``.
    """
    kp, vp, page_stride, pages, ps, hkv, d, cache_dt, dev = cache_fields(paged_kv_cache, kv_layout)
    dt = _row_dtype(append_key, d)
    if kv_scales is not None or cache_dt is FP8:
        scales = scale_fields(kv_scales, pages, ps, hkv, cache_dt, dev)
    elif dt is cache_dt:
        scales = _NO_SCALES
    else:
        raise ValueError(f"append_key dtype {dt} differs from the cache dtype {cache_dt}")
    nnz = append_key.shape[0]
    shape = (nnz, hkv, d)
    ks, vs = _rows(append_key, "append_key", shape, dt, dev), _rows(append_value, "append_value", shape, dt, dev)
    qshape = q.shape
    if len(qshape) != 3 or qshape[0] != nnz or qshape[2] != d:
        raise ValueError(f"q must be [{nnz}, Hq, {d}] in {dt}")
    qs = _rows(q, "q", qshape, dt, dev)
    qw = kw = err = 0
    wdt = dt
    if q_weight is not None:
        qw, wdt = _weight(q_weight, "q_weight", d, dt, dev), q_weight.dtype
    if k_weight is not None:
        kw = _weight(k_weight, "k_weight", d, dt, dev)
        if qw and k_weight.dtype is not wdt:
            raise ValueError("q_weight and k_weight must share one dtype")
        wdt = k_weight.dtype
    cdt, cst, cs_shape = cos.dtype, cos.stride(), cos.shape
    if cs_shape != (nnz, d) or sin.shape != cs_shape or sin.stride() != cst or cst[1] != 1 or sin.dtype is not cdt or \
            (cdt is not dt and cdt is not torch.float32):
        raise ValueError(f"cos and sin must both be [{nnz}, {d}] in {dt} or float32, with one row stride and a unit inner one")
    if cos.device != dev or sin.device != dev:
        raise ValueError(f"cos and sin are on {cos.device} and {sin.device}, the cache on {dev}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    bi, po = _ids(batch_indices, "batch_indices", dev), _ids(positions, "positions", dev)
    if batch_indices.numel() < nnz or positions.numel() < nnz:
        raise ValueError("q, append_key, append_value, batch_indices and positions disagree on nnz")
    idx, ptr, batch = _ids(kv_indices, "kv_indices", dev), _ids(kv_indptr, "kv_indptr", dev), kv_indptr.numel() - 1
    if batch < 0:
        raise ValueError("kv_indptr must have batch+1 entries")
    if err_count is not None:
        err = _ids(err_count, "err_count", dev)
    if q_out is None:
        q_out = torch.empty_like(q) if q.is_contiguous() else torch.empty(qshape, dtype=dt, device=dev)
        os = q_out.stride()
    else:
        os = _rows(q_out, "q_out", qshape, dt, dev)
    if nnz == 0:
        return q_out
    code = DTYPE_CODE[dt]
    check(call(CALL_NORM_ROPE, q.data_ptr(), qs[0], qs[1], q_out.data_ptr(), os[0], os[1], qshape[1], append_key.data_ptr(),
               ks[0], ks[1], append_value.data_ptr(), vs[0], vs[1], qw, kw, DTYPE_CODE[wdt], eps, cos.data_ptr(), sin.data_ptr(),
               cst[0], DTYPE_CODE[cdt], bi, po, nnz, kp, vp, page_stride, pages, *scales, idx, kv_indices.numel(), ptr, batch,
               hkv, d, ps, code, err, stream_ptr(dev)), "append_paged_kv_cache_with_norm_rope")
    return q_out


_NO_SCALES = (0, 0, 0)


def _weight(t, name: str, d: int, dt: torch.dtype, dev: torch.device) -> int:
    if not isinstance(t, torch.Tensor) or t.shape != (d,) or not t.is_contiguous() or (t.dtype is not dt and t.dtype is not torch.float32):
        raise ValueError(f"{name} must be [{d}] in {dt} or float32, contiguous")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the cache on {dev}")
    return t.data_ptr()


def read_paged_kv_cache(paged_kv_cache: CacheT, kv_scales, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                        dtype: torch.dtype, out: torch.Tensor | None = None, kv_layout: str = "NHD") -> torch.Tensor:
    """An 8-bit cache's listed pages in fp16, bf16 or fp32: page i of the result ``[len(kv_indices), 2,
    page_size, Hkv, D]`` holds the values of page ``kv_indices[i]``, for i < ``kv_indptr[-1]``, so with the
    page ids 0, 1, 2, ... it stands for the cache wherever one of ``dtype`` is read (the prefill wrapper does
    this by itself).  bf16 and fp32 hold every value exactly, fp16 those in its range.  Whole pages are
    read, with the slots past a sequence's end; an id outside the pool gives zeros; pages of ``out`` past
    the list are left as they were.  head_dim must be a multiple of 16, up to 512.
    """
    kp, vp, page_stride, pages, ps, hkv, d, cache_dt, dev = cache_fields(paged_kv_cache, kv_layout)
    scales = scale_fields(kv_scales, pages, ps, hkv, cache_dt, dev)
    if d % 16 or not 0 < d <= 512:
        raise ValueError("head_dim must be a multiple of 16, up to 512")
    idx, ptr, batch = _ids(kv_indices, "kv_indices", dev), _ids(kv_indptr, "kv_indptr", dev), kv_indptr.numel() - 1
    if batch < 0:
        raise ValueError("kv_indptr must have batch+1 entries")
    code = dtype_code(dtype)
    n = kv_indices.numel()
    shape = (n, 2, ps, hkv, d)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    elif out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be {list(shape)} in {dtype}, contiguous, on the cache's device")
    if n == 0 or batch == 0:
        return out
    check(call(CALL_READ_FP8, kp, vp, page_stride, pages, *scales, idx, n, ptr, batch, hkv, d, ps, out.data_ptr(), code,
               stream_ptr(dev)), "read_paged_kv_cache")
    return out
