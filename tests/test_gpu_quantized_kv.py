"""The quantised paged cache against its definition in 64 bits: every byte of
what is written, what stays untouched, and what is read back."""
import math

import pytest
import torch

import paged_reference as R
from lightserve_b200.kernels import (dequantize_kv_cache, quantize_kv_cache, quantized_kv_cache, rope_quantize_kv,
                                     rope_kv_write_slots)
from lightserve_b200.kernels.paged_attention import rope_kv_write

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _cache(nb, H, bs, D, fill=0xA5):
    c = quantized_kv_cache(nb, H, bs, D)
    for t in c:
        t.view(torch.uint8).fill_(fill)
    return c


def _cells(t, slots, bs):
    return t.view(torch.uint8)[slots // bs, :, slots % bs]


def _check_rows(cache, scale, slots, bs, x):
    """Bytes and scales at the slots are those of rows x [T, H, D]."""
    q, e = R.quantise(x.cpu())
    got = _cells(cache, slots, bs).view(torch.float8_e4m3fn).double().cpu()
    assert torch.equal(R.e8m0(_cells(scale, slots, bs)).cpu(), e)
    assert bool(((got == q) | (got.isnan() & q.isnan())).all())


def _values(T, H, D, dtype, g):
    x = torch.randn(T, H, D, generator=g) * torch.exp(2 * torch.randn(T, H, 1, generator=g))
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,D,bs", [(1, 1, 64, 16), (37, 3, 128, 16), (130, 2, 256, 32), (5, 4, 32, 8), (9, 1, 80, 16),
                                      (3, 2, 1, 4), (6, 5, 33, 1), (1000, 16, 128, 16)])
def test_written_and_read_back(T, H, D, bs, dtype):
    g = torch.Generator().manual_seed(T)
    nb = -(-T // bs) + 2
    k, v = (_values(T, H, D, dtype, g) for _ in range(2))
    slots = torch.randperm(nb * bs, generator=g)[:T].cuda()
    c = _cache(nb, H, bs, D)
    quantize_kv_cache(k, v, *c, slots)
    for cache, scale, x in ((c[0], c[2], k), (c[1], c[3], v)):
        _check_rows(cache, scale, slots, bs, x)
    for t in c:  # every other cell is as it was
        raw = t.view(torch.uint8).clone()
        raw[slots // bs, :, slots % bs] = 0xA5
        assert bool((raw == 0xA5).all())
    for out_type in TYPES:
        ko, vo = dequantize_kv_cache(*c, slots, out_type)
        most = torch.finfo(out_type).max
        for o, x in ((ko, k), (vo, v)):
            q, e = R.quantise(x.cpu())
            want = (q * e[..., None]).clamp(-most, most)
            # exact where the type holds the value; fp16 may round what lies below its normal range
            ok = (o.double().cpu() - want).abs() <= (2.0 ** -25 if out_type == torch.float16 else 0.0)
            assert bool(ok.all())


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values(dtype):
    """Zeros, one value, the type's largest, its smallest, ties, NaN and infinities."""
    D, top = 128, torch.finfo(dtype).max
    rows = torch.zeros(12, 1, D)
    rows[1, 0, 5] = 3.0
    rows[2, 0, :2] = torch.tensor([top, -top])
    rows[3, 0, :3] = torch.tensor([torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 8, 0.0])
    rows[4, 0, :16] = 256 + 16.0 * torch.arange(16)        # halfway cases of the top binade
    rows[5, 0, 0], rows[5, 0, 1] = 448.0, 449.0              # just over the border of two scales
    rows[6, 0, 0] = 448.0
    rows[7, 0, :3] = torch.tensor([math.nan, 1.0, -2.0])
    rows[8, 0, :4] = torch.tensor([math.inf, -math.inf, 0.5, 7.0])
    rows[9] = math.nan
    rows[10, 0] = torch.linspace(-1, 1, D) * 2.0 ** -9
    rows[10, 0, 0] = 448.0                                   # the rest falls into e4m3's subnormals
    rows[11, 0] = -0.0
    x = rows.to(dtype).cuda()
    slots = torch.arange(12).cuda()
    c = _cache(1, 1, 16, D)
    quantize_kv_cache(x, x, *c, slots)
    _check_rows(c[0], c[2], slots, 16, x)
    _check_rows(c[1], c[3], slots, 16, x)
    k, _ = dequantize_kv_cache(*c, slots, dtype)
    assert bool(k[9].isnan().all()) and bool(k[8, 0, :2].isnan().all()) and bool(k[8, 0, 2:].isfinite().all())
    assert bool(k[2].isfinite().all()) and float(k[2, 0, 0]) > 0.9 * top


def test_slots_outside_are_skipped_and_read_as_zero():
    T, H, D, bs, nb = 6, 2, 64, 16, 2
    k, v = (torch.randn(T, H, D, device="cuda") for _ in range(2))
    slots = torch.tensor([-1, 3, nb * bs, 31, -2 ** 40, 2 ** 40]).cuda()
    c = _cache(nb, H, bs, D)
    quantize_kv_cache(k, v, *c, slots)
    inside = torch.tensor([3, 31]).cuda()
    _check_rows(c[0], c[2], inside, bs, k[[1, 3]])
    assert int((c[2].view(torch.uint8) != 0xA5).sum()) <= 2 * H
    ko, vo = dequantize_kv_cache(*c, slots, torch.float32, k_out=torch.full((T, H, D), 5.0, device="cuda"))
    for t in (0, 2, 4, 5):
        assert bool((ko[t] == 0).all()) and bool((vo[t] == 0).all())
    again, _ = dequantize_kv_cache(*c, inside[[0, 0, 1]], torch.float32)
    assert torch.equal(again[0], again[1]) and torch.equal(again[0], ko[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows(dtype):
    """k and v as views of a fused projection, aligned and not."""
    T, H, D, bs = 19, 2, 64, 16
    for off in (0, 1, 8):
        wide = torch.randn(T, 3, H, D + 8, device="cuda").to(dtype)
        k, v = wide[:, 1, :, off:off + D], wide[:, 2, :, off:off + D]
        slots = torch.randperm(32, device="cuda")[:T]
        c = _cache(2, H, bs, D)
        quantize_kv_cache(k, v, *c, slots)
        _check_rows(c[0], c[2], slots, bs, k)
        _check_rows(c[1], c[3], slots, bs, v)


def _tables(D, dtype, far=96):
    a = torch.outer(torch.arange(far).double(), 10000.0 ** -(torch.arange(D // 2).double() / max(1, D // 2)))
    return tuple(torch.cat([t, t], -1).to(dtype).cuda().contiguous() for t in (a.cos(), a.sin()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,D,off", [(1, 1, 64, 0), (64, 16, 128, 0), (33, 3, 256, 0), (7, 2, 32, 0), (5, 2, 80, 0),
                                       (5, 2, 128, 3), (9, 1, 2, 0)])
def test_rope_form_equals_rope_then_quantise(T, H, D, off, dtype):
    """q, k_out and the cached rows are those of the 16-bit rotary write followed by quantisation, bit for bit,
    in the slot form and in the block-table form."""
    bs, mb = 16, 6
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(T, 3, H, D + off, generator=g).to(dtype).cuda()[..., off:]
    cos, sin = _tables(D, dtype)
    pos = torch.randint(0, 96, (T,), generator=g).cuda()
    nb = T * mb
    bt = torch.randperm(nb, generator=g).view(T, mb).to(torch.int32).cuda()
    if T > 4:
        bt[2] = -1
    ids = bt.gather(1, (pos // bs).unsqueeze(1)).squeeze(1).long()
    slots = torch.where(ids >= 0, ids * bs + pos % bs, ids)
    q_ref, k_ref = (torch.empty(T, H, D, dtype=dtype, device="cuda") for _ in range(2))
    plain = torch.zeros(nb, H, bs, D, dtype=dtype, device="cuda")
    rope_kv_write_slots(qkv, cos, sin, pos, slots, q_ref, k_ref, plain, plain.clone())
    want = _cache(nb, H, bs, D)
    quantize_kv_cache(k_ref, qkv[:, 2], *want, slots)
    for form in ({"slot_mapping": slots}, {"block_tables": bt}):
        got = _cache(nb, H, bs, D)
        q, k = torch.empty_like(q_ref), torch.empty_like(q_ref)
        cl = torch.full((T,), -7, dtype=torch.int32, device="cuda")
        rope_quantize_kv(qkv, cos, sin, pos, q, *got, context_lens=cl, k_out=k, **form)
        assert torch.equal(q, q_ref) and torch.equal(k, k_ref)
        assert torch.equal(cl.long(), pos + 1)
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("D", [64, 80])
def test_rope_positions_outside_the_table(D):
    T, H, bs = 5, 2, 16
    qkv = torch.randn(T, 3, H, D, device="cuda")
    cos, sin = _tables(D, torch.float32)
    pos = torch.tensor([-1, 96, 4, 2 ** 40, 95]).cuda()
    bt = torch.arange(T * 6, dtype=torch.int32).view(T, 6).cuda()
    c = _cache(T * 6, H, bs, D)
    q = torch.zeros(T, H, D, device="cuda")
    cl = torch.full((T,), 9, dtype=torch.int32, device="cuda")
    rope_quantize_kv(qkv, cos, sin, pos, q, *c, block_tables=bt, context_lens=cl)
    assert cl.tolist() == [0, 0, 5, 0, 96]
    assert bool(q[[0, 1, 3]].isnan().all()) and bool(q[[2, 4]].isfinite().all())
    assert int((c[2].view(torch.uint8) != 0xA5).sum()) <= 2 * H and int((c[0].view(torch.uint8) != 0xA5).any(-1).sum()) <= 2 * H


def test_captured_and_on_another_stream():
    T, H, D, bs = 40, 2, 128, 16
    k, v = (torch.randn(T, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    slots = torch.randperm(64, device="cuda")[:T]
    c = _cache(4, H, bs, D)
    out = torch.empty(2, T, H, D, dtype=torch.bfloat16, device="cuda")
    quantize_kv_cache(k, v, *c, slots)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        quantize_kv_cache(k, v, *c, slots)
        dequantize_kv_cache(*c, slots, torch.bfloat16, k_out=out[0], v_out=out[1])
    for i in range(3):
        k.copy_(torch.randn(T, H, D).to(torch.bfloat16) * (i + 1))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        _check_rows(c[0], c[2], slots, bs, k)
        q, e = R.quantise(k.cpu())
        assert torch.equal(out[0].double().cpu(), q * e[..., None])


def test_offsets_past_32_bits():
    H, bs, D, T = 16, 16, 128, 50
    nb = 2 ** 32 // (H * bs * D) + 8
    k, v = (torch.randn(T, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    cells = (nb, H, bs)
    c = [torch.empty(*cells, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    c += [torch.empty(cells, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    slots = (nb * bs - 1 - torch.arange(T)).cuda()
    quantize_kv_cache(k, v, *c, slots)
    _check_rows(c[0], c[2], slots, bs, k)
    _check_rows(c[1], c[3], slots, bs, v)
    ko, _ = dequantize_kv_cache(*c, slots, torch.bfloat16)
    q, e = R.quantise(k.cpu())
    assert torch.equal(ko.double().cpu(), q * e[..., None])
