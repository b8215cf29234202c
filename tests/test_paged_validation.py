"""Refusals of the paged-cache operators, each by its own message, before
anything is launched (CPU tensors; the C entries with null pointers)."""
import pytest
import torch

import paged_reference as R
from lightserve_b200 import _lib
from lightserve_b200.kernels import (dequantize_kv_cache, paged_chunk_attention, paged_chunk_workspace,
                                     paged_decode_attention, quantize_kv_cache, quantized_kv_cache, rope_quantize_kv)

BF16 = torch.bfloat16


def _chunk(quantised=False, **kw):
    b = R.build([40, 9], [5, 2], 2, 2, 64, 16, BF16, quantised=quantised)
    args = dict(q=b["q"], k_cache=b["k_cache"], v_cache=b["v_cache"], block_tables=b["block_tables"],
                context_lens=b["context_lens"], cu_seqlens_q=b["cu"], max_seqlen_q=5, k_scale=b["k_scale"],
                v_scale=b["v_scale"])
    args.update({k: (v(args) if callable(v) else v) for k, v in kw.items()})
    return paged_chunk_attention(**args)


@pytest.mark.parametrize("match,change", [
    ("T, H, D", {"q": lambda a: a["q"][0]}),
    ("num_blocks, H, block_size, D", {"k_cache": lambda a: a["k_cache"][0]}),
    ("contiguous", {"k_cache": lambda a: a["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)}),
    ("dtype mismatch", {"k_cache": lambda a: a["k_cache"].half()}),
    ("dtypes must match", {"k_cache": lambda a: a["k_cache"].half(), "v_cache": lambda a: a["v_cache"].half()}),
    ("head dim", {"q": lambda a: a["q"][..., :32]}),
    ("no multiple", {"q": lambda a: a["q"][:, :3]}),
    ("unsupported dtype|dtypes must match", {"q": lambda a: a["q"].double()}),
    ("along D", {"q": lambda a: a["q"].transpose(1, 2).contiguous().transpose(1, 2)}),
    ("block_tables", {"block_tables": lambda a: a["block_tables"].long()}),
    ("block_tables", {"block_tables": lambda a: a["block_tables"].t().contiguous().t()}),
    ("context_lens", {"context_lens": lambda a: a["context_lens"][:1]}),
    ("context_lens", {"context_lens": lambda a: a["context_lens"].long()}),
    ("cu_seqlens_q must be", {"cu_seqlens_q": lambda a: a["cu_seqlens_q"][:2]}),
    ("cu_seqlens_q is required", {"cu_seqlens_q": None}),
    ("max_seqlen_q", {"max_seqlen_q": 8}),
    ("max_seqlen_q", {"max_seqlen_q": -1}),
    ("window must be positive", {"window": 0}),
    ("window must be positive", {"window": -3}),
    ("num_sinks must not be negative", {"window": 4, "num_sinks": -1}),
    ("needs a window", {"num_sinks": 4}),
    ("go together", {"k_scale": torch.zeros(1)}),
    ("lse", {"lse": torch.zeros(4, 6)}),
    ("CUDA", {}),
])
def test_chunk_refuses(match, change):
    with pytest.raises(AssertionError, match=match):
        _chunk(**change)


@pytest.mark.parametrize("match,change", [
    ("float8_e4m3fn", {"k_cache": lambda a: a["k_cache"].float(), "v_cache": lambda a: a["v_cache"].float()}),
    ("dtypes must match", {"k_scale": None, "v_scale": None}),
    ("float8_e8m0fnu", {"k_scale": lambda a: a["k_scale"].view(torch.uint8)}),
    ("num_blocks, H, block_size", {"k_scale": lambda a: a["k_scale"][:, :1], "v_scale": lambda a: a["v_scale"][:, :1]}),
    ("CUDA", {}),
])
def test_quantised_chunk_refuses(match, change):
    with pytest.raises(AssertionError, match=match):
        _chunk(True, **change)


def test_page_size_must_be_a_power_of_two():
    b = R.build([40], [5], 2, 1, 64, 12, BF16)
    with pytest.raises(AssertionError, match="power of two"):
        paged_chunk_attention(b["q"], b["k_cache"], b["v_cache"], b["block_tables"], b["context_lens"], b["cu"], 5)


def test_decode_refuses():
    b = R.build([40, 9], [1, 1], 2, 2, 64, 16, BF16)
    args = (b["q"], b["k_cache"], b["v_cache"], b["block_tables"], b["context_lens"])
    with pytest.raises(AssertionError, match="CUDA"):
        paged_decode_attention(*args)
    with pytest.raises(AssertionError, match="no multiple"):
        paged_decode_attention(b["q"][:, :3], *args[1:])
    with pytest.raises(AssertionError, match="one row"):
        paged_decode_attention(b["q"][:1], *args[1:])
    with pytest.raises(AssertionError, match="needs a window"):
        paged_decode_attention(*args, num_sinks=3)


def _store(**kw):
    c = quantized_kv_cache(4, 2, 16, 64, device="cpu")
    x = torch.randn(7, 2, 64)
    args = dict(k=x, v=x.clone(), k_cache=c[0], v_cache=c[1], k_scale=c[2], v_scale=c[3], slot_mapping=torch.arange(7))
    args.update({k: (v(args) if callable(v) else v) for k, v in kw.items()})
    return quantize_kv_cache(**args)


@pytest.mark.parametrize("match,change", [
    ("T, H, D", {"v": lambda a: a["v"][:3]}),
    ("dtype mismatch", {"v": lambda a: a["v"].half()}),
    ("needs its scales", {"k_scale": None, "v_scale": None}),
    ("float8_e4m3fn", {"k_cache": lambda a: a["k_cache"].float(), "v_cache": lambda a: a["v_cache"].float()}),
    ("heads/dim", {"k": lambda a: a["k"][..., :32], "v": lambda a: a["v"][..., :32]}),
    ("along D", {"k": lambda a: a["k"].transpose(1, 2).contiguous().transpose(1, 2)}),
    ("slot_mapping", {"slot_mapping": torch.arange(7, dtype=torch.int32)}),
    ("slot_mapping", {"slot_mapping": torch.arange(6)}),
    ("unsupported dtype", {"k": lambda a: a["k"].double(), "v": lambda a: a["v"].double()}),
    ("CUDA", {}),
])
def test_quantize_refuses(match, change):
    with pytest.raises(AssertionError, match=match):
        _store(**change)


def test_dequantize_refuses():
    c = quantized_kv_cache(4, 2, 16, 64, device="cpu")
    for match, args, kw in (("unsupported dtype", (torch.arange(3), torch.float64), {}),
                            ("slot_mapping", (torch.arange(3).int(), BF16), {}),
                            ("outputs", (torch.arange(3), BF16), {"k_out": torch.empty(3, 2, 64)}),
                            ("CUDA", (torch.arange(3), BF16), {})):
        with pytest.raises(AssertionError, match=match):
            dequantize_kv_cache(*c, *args, **kw)


def _rope(**kw):
    c = quantized_kv_cache(4, 2, 16, 64, device="cpu")
    args = dict(qkv=torch.randn(7, 3, 2, 64), cos=torch.ones(32, 64), sin=torch.ones(32, 64), positions=torch.arange(7),
                q_out=torch.empty(7, 2, 64), k_cache=c[0], v_cache=c[1], k_scale=c[2], v_scale=c[3],
                slot_mapping=torch.arange(7))
    args.update({k: (v(args) if callable(v) else v) for k, v in kw.items()})
    return rope_quantize_kv(**args)


@pytest.mark.parametrize("match,change", [
    ("qkv must be", {"qkv": lambda a: a["qkv"][:, :2]}),
    ("tables", {"cos": lambda a: a["cos"][:, :32]}),
    ("share a dtype", {"q_out": lambda a: a["q_out"].half()}),
    ("positions", {"positions": torch.arange(7).int()}),
    ("not both", {"slot_mapping": None}),
    ("not both", {"block_tables": torch.zeros(7, 2, dtype=torch.int32)}),
    ("block_tables", {"slot_mapping": None, "block_tables": torch.zeros(6, 2, dtype=torch.int32)}),
    ("CUDA", {}),
])
def test_rope_refuses(match, change):
    with pytest.raises(AssertionError, match=match):
        _rope(**change)


def test_c_entries_refuse_without_launching():
    lib = _lib.load()

    def attn(S=1, T=1, most=1, Hq=2, Hkv=1, D=64, mb=4, bs=16, nb=8, window=0, sinks=0, dtype=1, kv=1, impl=0, ptr=None):
        return lib.lsb_paged_attn(ptr, ptr, ptr, None, None, ptr, ptr, None, ptr, None, S, T, most, Hq, Hkv, D, mb, bs,
                                  nb, Hq * D, D, Hq * D, D, window, sinks, 1.0, dtype, kv, impl, None, 0, None)

    for match, kw in (("bad sizes", {"D": 0}), ("bad sizes", {"S": -1}), ("no multiple", {"Hq": 3, "Hkv": 2}),
                      ("power of two", {"bs": 12}), ("unsupported dtype", {"dtype": 9, "kv": 9}),
                      ("e4m3", {"kv": 2}), ("neither is negative", {"window": -1}), ("need a window", {"sinks": 1}),
                      ("above total_q", {"most": 2}), ("one row", {"T": 2}), ("null pointer", {}),
                      ("scales", {"kv": 3, "ptr": 16}), ("too large", {"mb": 1 << 40, "ptr": 16}),
                      ("bad impl", {"impl": 77, "ptr": 16}), ("workspace", {"mb": 1 << 12, "ptr": 16})):
        assert attn(**kw) == _lib.LSB_ERR_INVALID, kw
        assert match in _lib.last_error(), (match, _lib.last_error())
    assert attn(D=264, ptr=16) == _lib.LSB_ERR_UNSUPPORTED and "head dim" in _lib.last_error()
    assert attn(S=0, T=0, most=0) == _lib.LSB_OK
    for rc in (lib.lsb_kv_quantize(*[None] * 7, 1, 1, 0, 1, 1, 0, 0, 0, 0, 1, None),
               lib.lsb_kv_quantize(*[None] * 7, 1, 1, 64, 1, 1, 0, 0, 0, 0, 1, None),
               lib.lsb_kv_quantize(*[None] * 7, 1 << 31, 1, 64, 1, 1, 0, 0, 0, 0, 1, None),
               lib.lsb_kv_dequantize(*[None] * 7, 1, 1, 64, 1, 1, 9, None),
               lib.lsb_kv_dequantize(*[None] * 7, 1, 1, 64, 1, 1, 1, None),
               lib.lsb_rope_kv_quantize(None, 0, 0, 0, None, None, 0, 8, None, None, None, 0, *[None] * 7, 1, 1, 64, 1, 1,
                                        1, None),
               lib.lsb_rope_kv_quantize(None, 0, 0, 0, None, None, 0, 8, None, 16, None, 0, *[None] * 7, 1, 1, 63, 1, 1,
                                        1, None)):
        assert rc == _lib.LSB_ERR_INVALID
    assert lib.lsb_kv_quantize(*[None] * 7, 0, 1, 64, 1, 1, 0, 0, 0, 0, 1, None) == _lib.LSB_OK


def test_workspace_follows_the_window():
    """A window bounds the keys a row can see, and so the ranges they are split into."""
    full = paged_chunk_workspace((1, 8, 128), 1, 1, 8, 4096, 16, "cpu")
    short = paged_chunk_workspace((1, 8, 128), 1, 1, 8, 4096, 16, "cpu", 64, 4)
    many = paged_chunk_workspace((70000, 8, 128), 8, 65536, 8, 4096, 16, "cpu")
    assert full.numel() > short.numel() > many.numel() == 1


@pytest.mark.parametrize("window,sinks", [(1 << 62, 1 << 62), (1 << 70, 0), (64, 1 << 62), (1 << 62, 3)])
def test_workspace_of_windows_past_every_position(window, sinks):
    """Sizes whose sum leaves 64 bits still ask for the scratch of the whole context."""
    full = paged_chunk_workspace((1, 8, 128), 1, 1, 8, 4096, 16, "cpu")
    assert paged_chunk_workspace((1, 8, 128), 1, 1, 8, 4096, 16, "cpu", window, sinks).numel() == full.numel()
    raw = min(window, (1 << 63) - 1), sinks
    assert _lib.load().lsb_paged_attn_workspace_size(1, 1, 1, 8, 8, 128, 4096, 16, *raw) == 4 * full.numel()
