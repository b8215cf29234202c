"""Quantised paged KV cache: e4m3 rows, one power-of-two scale per (token, head).

A cache of half the bytes of the 16-bit one behind the same block tables and
slots: ``k_cache, v_cache`` are ``float8_e4m3fn [num_blocks, H, block_size, D]``
and ``k_scale, v_scale`` ``float8_e8m0fnu [num_blocks, H, block_size]``. A row x
is stored with the smallest power of two s that takes its largest finite
magnitude to 448 or less, as e4m3(x / s) rounded to nearest even: within 2^-4
of each value, or 2^-10 s for values below 2^-6 s. The product e4m3 * s is
exact in the model dtype (held at its largest finite value where the rounding
went past it). NaN and infinities are stored as NaN. lightserve's cache has no
quantised form (``engine/config.py:7-11`` leaves the layout to the deployment).

``quantize_kv_cache`` and ``rope_quantize_kv`` write rows, ``dequantize_kv_cache``
reads them back, and ``paged_decode_attention`` and ``paged_chunk_attention``
attend over them. Computation: ``lsb_kv_quantize``, ``lsb_rope_kv_quantize`` and
``lsb_kv_dequantize`` in liblightserve_b200.so.
"""
from __future__ import annotations

import torch

from .. import _lib
from .paged_chunk_attention import _check_cache


def quantized_kv_cache(num_blocks: int, num_heads: int, block_size: int, head_dim: int, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of an empty quantised cache (zeros)."""
    cell = (num_blocks, num_heads, block_size)
    rows = [torch.zeros(*cell, head_dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
            for _ in range(2)]
    scales = [torch.zeros(cell, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu) for _ in range(2)]
    return (*rows, *scales)


def _check_slots(slot_mapping, T, index):
    assert slot_mapping.dtype == torch.int64 and slot_mapping.shape == (T,) and slot_mapping.is_contiguous(), (
        "slot_mapping must be a contiguous int64 [T]")
    assert slot_mapping.get_device() == index, "tensors must be on one device"


def quantize_kv_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """``write_kv_cache`` into a quantised cache: rows ``k[t], v[t]`` (``[T, H, D]``,
    fp32/bf16/fp16) go to slot ``slot_mapping[t]`` (``block_id * block_size +
    offset``; slots outside the cache, such as -1, are skipped). The slots of one
    call must differ: two tokens in one slot leave it with bytes of either."""
    shape, dtype, index = k.shape, k.dtype, k.get_device()
    assert len(shape) == 3 and shape == v.shape, f"k/v must be [T, H, D], got {tuple(shape)}/{tuple(v.shape)}"
    T, H, D = shape
    assert dtype == v.dtype, f"dtype mismatch: k={dtype} v={v.dtype}"
    assert k_scale is not None and v_scale is not None, "a quantised cache needs its scales"
    (nb, Hc, bs, Dc), _ = _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, index)
    assert Hc == H and Dc == D, f"cache heads/dim {(Hc, Dc)} do not match k {(H, D)}"
    code = _lib.dtype_code(dtype)
    assert v.get_device() == index, "tensors must be on one device"
    sk, sv = k.stride(), v.stride()
    assert sk[2] == 1 and sv[2] == 1, "k/v must be contiguous along D"
    _check_slots(slot_mapping, T, index)
    assert index >= 0, "lightserve_b200 kernels need CUDA tensors"
    if T == 0 or H == 0 or D == 0:
        return
    assert nb > 0, "empty cache"
    lib, device = _lib.load(), k.device
    with _lib.device_guard(device):
        rc = lib.lsb_kv_quantize(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), slot_mapping.data_ptr(), T, H, D, nb, bs, sk[0], sk[1], sv[0], sv[1], code,
            _lib.stream_ptr(device),
        )
    _lib.check(rc, "lsb_kv_quantize")


def dequantize_kv_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype,
                        k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
    """Rows of a quantised cache by slot, as ``(k, v)`` of ``[T, H, D]`` in ``dtype``
    (fp32/bf16/fp16), written into ``k_out``/``v_out`` when given. Slots outside
    the cache give zeros; a slot may be read more than once."""
    assert k_scale is not None and v_scale is not None, "a quantised cache needs its scales"
    code, index = _lib.dtype_code(dtype), k_cache.get_device()
    (nb, H, bs, D), _ = _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, index)
    assert slot_mapping.ndim == 1, "slot_mapping must be a contiguous int64 [T]"
    T = slot_mapping.shape[0]
    _check_slots(slot_mapping, T, index)
    for o in (k_out, v_out):
        assert o is None or (o.shape == (T, H, D) and o.dtype == dtype and o.get_device() == index
                             and o.is_contiguous()), (
            f"outputs must be contiguous {dtype} [T, H, D] on the cache's device")
    assert index >= 0, "lightserve_b200 kernels need CUDA tensors"
    device = k_cache.device
    if k_out is None:
        k_out = torch.empty(T, H, D, dtype=dtype, device=device)
    if v_out is None:
        v_out = torch.empty(T, H, D, dtype=dtype, device=device)
    if T == 0 or H == 0 or D == 0:
        return k_out, v_out
    assert nb > 0, "empty cache"
    lib = _lib.load()
    with _lib.device_guard(device):
        rc = lib.lsb_kv_dequantize(
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            slot_mapping.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), T, H, D, nb, bs, code,
            _lib.stream_ptr(device),
        )
    _lib.check(rc, "lsb_kv_dequantize")
    return k_out, v_out


def rope_quantize_kv(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                     q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     k_scale: torch.Tensor, v_scale: torch.Tensor, *,
                     slot_mapping: torch.Tensor | None = None, block_tables: torch.Tensor | None = None,
                     context_lens: torch.Tensor | None = None,
                     k_out: torch.Tensor | None = None) -> torch.Tensor:
    """``rope_kv_write`` / ``rope_kv_write_slots`` into a quantised cache: rotary
    embedding of q and k, rotated k and v quantised into the cache, in one launch.

    qkv: ``[T, 3, H, D]`` (the fused QKV projection); cos/sin: ``[max_pos, D]``
    tables in its dtype; positions: int64 ``[T]``. Each token's slot comes either
    from ``slot_mapping`` (int64 ``[T]``; a prompt's tokens) or from
    ``block_tables`` (int32 ``[T, max_blocks]``, one token per sequence; a decode
    step), exactly one of them; tokens whose slot lies outside the cache are not
    written, and the slots of one call must differ. Rotated q goes to ``q_out``
    and, when given, rotated k to ``k_out`` (``[T, H, D]`` contiguous), with the
    roundings of ``rope_kv_write``; ``context_lens`` (int32 ``[T]``) receives
    positions + 1. A position outside the tables gives NaN rows in ``q_out`` and
    ``k_out``, context length 0 and no cache write. Returns ``q_out``."""
    shape, sx, dtype, index = qkv.shape, qkv.stride(), qkv.dtype, qkv.get_device()
    assert len(shape) == 4 and shape[1] == 3 and sx[3] == 1, "qkv must be [T, 3, H, D]"
    T, _, H, D = shape
    assert D % 2 == 0, f"head dim {D} must be even"
    code = _lib.dtype_code(dtype)
    assert k_scale is not None and v_scale is not None, "a quantised cache needs its scales"
    (nb, Hc, bs, Dc), _ = _check_cache(k_cache, v_cache, k_scale, v_scale, dtype, index)
    assert Hc == H and Dc == D, f"cache heads/dim {(Hc, Dc)} do not match qkv {(H, D)}"
    table, st = cos.shape, cos.stride()
    assert len(table) == 2 and table == sin.shape and table[1] == D and st == sin.stride(), (
        "cos and sin must be [max_pos, D] tables of one layout")
    assert st[1] == 1 and table[0] > 0
    assert dtype == cos.dtype == sin.dtype == q_out.dtype, "qkv, tables and q_out must share a dtype"
    assert q_out.shape == (T, H, D) and q_out.is_contiguous()
    if k_out is not None:
        assert k_out.shape == (T, H, D) and k_out.is_contiguous() and k_out.dtype == dtype
        assert k_out.get_device() == index
    assert positions.dtype == torch.int64 and positions.shape == (T,) and positions.is_contiguous(), (
        "positions must be a contiguous int64 [T]")
    assert cos.get_device() == sin.get_device() == q_out.get_device() == positions.get_device() == index, (
        "tensors must be on one device")
    assert (slot_mapping is None) != (block_tables is None), "give slot_mapping or block_tables, not both"
    max_blocks = 0
    if slot_mapping is not None:
        _check_slots(slot_mapping, T, index)
    else:
        assert block_tables.dtype == torch.int32 and block_tables.ndim == 2 and block_tables.shape[0] == T, (
            "block_tables must be int32 [T, max_blocks]")
        max_blocks = block_tables.shape[1]
        assert block_tables.is_contiguous() and max_blocks > 0 and block_tables.get_device() == index
    if context_lens is not None:
        assert context_lens.dtype == torch.int32 and context_lens.shape == (T,) and context_lens.is_contiguous()
        assert context_lens.get_device() == index
    assert index >= 0, "lightserve_b200 kernels need CUDA tensors"
    if T == 0 or H == 0 or D == 0:
        return q_out
    assert nb > 0, "empty cache"
    lib, device = _lib.load(), qkv.device
    with _lib.device_guard(device):
        rc = lib.lsb_rope_kv_quantize(
            qkv.data_ptr(), sx[0], sx[1], sx[2], cos.data_ptr(), sin.data_ptr(), st[0], table[0],
            positions.data_ptr(), _lib.ptr(slot_mapping), _lib.ptr(block_tables), max_blocks, q_out.data_ptr(),
            _lib.ptr(k_out), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            _lib.ptr(context_lens), T, H, D, nb, bs, code, _lib.stream_ptr(device),
        )
    _lib.check(rc, "lsb_rope_kv_quantize")
    return q_out
