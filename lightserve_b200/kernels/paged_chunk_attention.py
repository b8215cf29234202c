"""Attention of new tokens over a paged KV cache.

``paged_chunk_attention`` is the step between ``flash_attention_varlen`` (a
whole prompt, K/V in hand) and ``paged_decode_attention`` (one token per
sequence): each sequence brings any number of new tokens, whose K/V are already
in the cache, and attends to everything it has cached. It serves a prompt
prefilled in chunks, a prompt behind a cached prefix, and drafted tokens
verified in one pass. lightserve has no such operator (``engine/request.py:86-93``
names the case); the cache is addressed through the block tables of
``engine/block_manager.py`` (``:58-61``), as ``paged_decode_attention`` does.

Computation: ``lsb_paged_attn`` in liblightserve_b200.so.
"""
from __future__ import annotations

import math

import torch

from .. import _lib


def _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, index):
    """Checks of a 16/32-bit cache of type ``dtype``, or of an e4m3 cache with
    its scales, on CUDA device ``index`` (-1: CPU); returns the cache's shape and
    C dtype code."""
    shape, kind = k_cache.shape, k_cache.dtype
    assert len(shape) == 4 and shape == v_cache.shape, "caches must be [num_blocks, H, block_size, D]"
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous"
    assert kind == v_cache.dtype, f"dtype mismatch: k_cache={kind} v_cache={v_cache.dtype}"
    assert (k_scale is None) == (v_scale is None), "k_scale and v_scale go together"
    if k_scale is None:
        assert kind == dtype, f"q/cache dtypes must match, got {dtype} and {kind}"
        code = _lib.dtype_code(dtype)
    else:
        assert kind == torch.float8_e4m3fn, f"scales go with a float8_e4m3fn cache, got {kind}"
        assert k_scale.dtype == v_scale.dtype == torch.float8_e8m0fnu, "scales must be float8_e8m0fnu"
        assert k_scale.shape == v_scale.shape == shape[:3], "scales must be [num_blocks, H, block_size]"
        assert k_scale.is_contiguous() and v_scale.is_contiguous(), "scales must be contiguous"
        assert k_scale.get_device() == v_scale.get_device() == index, "tensors must be on one device"
        code = _lib.DTYPE_E4M3
    assert k_cache.get_device() == v_cache.get_device() == index, "tensors must be on one device"
    bs = shape[2]
    assert bs > 0 and (bs & (bs - 1)) == 0, "block_size must be a power of two"
    return shape, code


def _window_args(window, num_sinks):
    """(window, num_sinks) as the C entry takes them (0: no window; both held at
    2^31, past every position)."""
    assert window is None or int(window) > 0, f"window must be positive, got {window}"
    assert int(num_sinks) >= 0, f"num_sinks must not be negative, got {num_sinks}"
    assert window is not None or not num_sinks, "num_sinks needs a window (without one every key is visible)"
    return min(int(window or 0), 1 << 31), min(int(num_sinks), 1 << 31)


def paged_chunk_workspace(q_shape, num_seqs: int, max_seqlen_q: int, num_kv_heads: int,
                          max_blocks_per_seq: int, block_size: int, device, window: int | None = None,
                          num_sinks: int = 0) -> torch.Tensor:
    """fp32 scratch for split key ranges (one element when none is needed)."""
    T, Hq, D = q_shape
    w, sinks = _window_args(window, num_sinks)
    nbytes = _lib.load().lsb_paged_attn_workspace_size(num_seqs, T, max_seqlen_q, Hq, num_kv_heads, D,
                                                       max_blocks_per_seq, block_size, w, sinks)
    return torch.empty(max(nbytes // 4, 1), dtype=torch.float32, device=device)


def _paged_attn(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, max_seqlen_q, window,
                num_sinks, k_scale, v_scale, scale, out, lse, workspace, impl=_lib.IMPL_AUTO):
    assert q.ndim == 3, f"q must be [T, H, D], got {q.ndim}D"
    T, Hq, D = shape = q.shape
    dtype, index, max_q = q.dtype, q.get_device(), int(max_seqlen_q)
    w, sinks = _window_args(window, num_sinks)
    (nb, Hkv, bs, Dc), kv_code = _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, index)
    assert Dc == D, f"cache head dim {Dc} does not match q's {D}"
    assert Hkv > 0 and Hq % Hkv == 0, f"{Hq} query heads are no multiple of the cache's {Hkv}"
    code = _lib.dtype_code(dtype)
    sq = q.stride()
    assert sq[2] == 1, "q must be contiguous along D"
    assert block_tables.dtype == torch.int32 and block_tables.ndim == 2 and block_tables.is_contiguous(), (
        "block_tables must be a contiguous int32 [num_seqs, max_blocks]")
    S, max_blocks = block_tables.shape
    assert context_lens.dtype == torch.int32 and context_lens.shape == (S,) and context_lens.is_contiguous(), (
        "context_lens must be a contiguous int32 [num_seqs]")
    assert block_tables.get_device() == context_lens.get_device() == index, "tensors must be on one device"
    if cu_seqlens_q is not None:
        assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_q.shape == (S + 1,), (
            "cu_seqlens_q must be int32 [num_seqs + 1]")
        assert cu_seqlens_q.is_contiguous() and cu_seqlens_q.get_device() == index
        assert 0 <= max_q <= T, f"max_seqlen_q {max_seqlen_q} outside [0, {T}]"
    else:
        assert S == T, f"one row of q per sequence: q has {T}, block_tables {S}"
    if lse is not None:
        assert lse.shape == (Hq, T) and lse.dtype == torch.float32 and lse.is_contiguous(), (
            "lse must be a contiguous float32 [H, T]")
        assert lse.get_device() == index
    assert index >= 0, "lightserve_b200 kernels need CUDA tensors"
    if out is None:
        out = torch.empty_like(q)
    else:
        assert out.shape == shape and out.dtype == dtype and out.get_device() == index
    so = out.stride()
    assert so[2] == 1, "out must be contiguous along D"
    if S == 0 or T == 0 or Hq == 0 or D == 0 or max_q == 0:
        return out
    assert max_blocks > 0 and nb > 0, "empty block table or cache"
    lib = _lib.load()
    if workspace is None:
        ws_bytes = lib.lsb_paged_attn_workspace_size(S, T, max_q, Hq, Hkv, D, max_blocks, bs, w, sinks)
        if ws_bytes:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    else:
        assert workspace.get_device() == index and workspace.is_contiguous()
        ws_bytes = workspace.numel() * workspace.element_size()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    device = q.device
    with _lib.device_guard(device):
        rc = lib.lsb_paged_attn(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scale), _lib.ptr(v_scale),
            block_tables.data_ptr(), context_lens.data_ptr(), _lib.ptr(cu_seqlens_q), out.data_ptr(),
            _lib.ptr(lse), S, T, max_q, Hq, Hkv, D, max_blocks, bs, nb, sq[0], sq[1], so[0], so[1], w, sinks,
            scale, code, kv_code, impl, _lib.ptr(workspace), ws_bytes, _lib.stream_ptr(device),
        )
    _lib.check(rc, "lsb_paged_attn")
    return out


def paged_chunk_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          block_tables: torch.Tensor, context_lens: torch.Tensor,
                          cu_seqlens_q: torch.Tensor, max_seqlen_q: int, *,
                          window: int | None = None, num_sinks: int = 0,
                          k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                          scale: float | None = None, out: torch.Tensor | None = None,
                          lse: torch.Tensor | None = None,
                          workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each sequence's new tokens over its cached keys.

    q: ``[T, Hq, D]`` packed along the token axis (any token/head strides);
    sequence s brings rows ``[cu_seqlens_q[s], cu_seqlens_q[s+1])`` (int32
    ``[num_seqs + 1]``, non-decreasing), at most ``max_seqlen_q`` of them; an
    empty range is allowed. k_cache, v_cache: ``[num_blocks, Hkv, block_size, D]``
    in q's dtype, or e4m3 with ``k_scale``/``v_scale`` (see
    ``quantize_kv_cache``); Hq is a multiple of Hkv, query head h reading cache
    head ``h // (Hq // Hkv)``. block_tables: int32 ``[num_seqs, max_blocks]``;
    context_lens: int32 ``[num_seqs]``, the cached tokens *including* the new
    ones, whose K/V the caller has written.

    The i-th of n new tokens stands at position ``p = context_lens - n + i`` and
    sees key j when ``j <= p`` and, with ``window``, when ``p - j < window`` or
    ``j < num_sinks`` (the token itself counts as one of the window). Block ids
    outside the cache (such as -1) hold no keys, so pages that have left the
    window may be freed. A row that sees no key gives 0 (``lse`` -inf). Cached
    values that no row of a sequence sees (past the context, before the window)
    are never used, whatever they hold; a NaN or infinity at a key that one row
    sees may reach the other new rows of its sequence. Sums are fp32 and
    divided at the end: values times the number of keys stay below 2^119. Key
    ranges are cut by the table's width: one much wider than its contexts is slower.

    Rows of q that belong to no sequence, or lie past ``max_seqlen_q`` of
    theirs, are not computed: their rows of ``out`` stay as they were. ``lse``
    (fp32 ``[Hq, T]``) receives the log-sum-exp of the scaled scores. scale
    defaults to ``1/sqrt(D)``; D is at most 256. With ``out`` and ``workspace``
    (``paged_chunk_workspace``) the call allocates nothing and can be captured
    into a CUDA graph; calls that run at the same time need workspaces of
    their own."""
    assert cu_seqlens_q is not None, "cu_seqlens_q is required"
    return _paged_attn(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, max_seqlen_q,
                       window, num_sinks, k_scale, v_scale, scale, out, lse, workspace)
