"""Weights and values at the ends of their ranges in attention over a paged cache, by every kernel."""
import math

import pytest
import torch

import paged_reference as R
from lightserve_b200 import _lib
from lightserve_b200.kernels.paged_chunk_attention import _paged_attn

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
IMPLS = {"auto": _lib.IMPL_AUTO, "simt": _lib.IMPL_SIMT, "rows": _lib.IMPL_ROWS, "tc": _lib.IMPL_TCGEN05}


def _scored(keys, value, new, D, dtype, quantised):
    """One sequence whose key j has the score keys[j] * scale with every row: q is 1 in the first channel, K is keys
    there. value [ctx]: its V in all channels. Keys and values must be exact in dtype (and e4m3 with their scale)."""
    ctx, bs = len(keys), 16
    b = R.build([ctx], [new], 1, 1, D, bs, dtype, garbage=False, seed=61)
    b["q"].zero_()
    b["q"][..., 0] = 1
    at = b["block_tables"][0].long()[torch.arange(ctx) // bs], 0, torch.arange(ctx) % bs
    k, v = (torch.zeros(b[n].shape, dtype=torch.float64) for n in ("k_cache", "v_cache"))
    k[(*at, 0)] = torch.as_tensor(keys, dtype=torch.float64)
    v[at] = torch.as_tensor(value, dtype=torch.float64)[:, None]
    b |= {"k_cache": k.to(dtype), "v_cache": v.to(dtype)}
    if quantised:
        (kq, ks), (vq, vs) = (R.quantise(b[n]) for n in ("k_cache", "v_cache"))
        b |= {"k_cache": kq.float().to(torch.float8_e4m3fn), "v_cache": vq.float().to(torch.float8_e4m3fn),
              "k_scale": ks.float().to(torch.float8_e8m0fnu), "v_scale": vs.float().to(torch.float8_e8m0fnu)}
    return b


def _run(b, scale, impl):
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}
    lse = torch.full((1, b["q"].shape[0]), 7.0, device="cuda")
    out = _paged_attn(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"], b["most"],
                      None, 0, c["k_scale"], c["v_scale"], scale, None, lse, None, IMPLS[impl])
    return out, lse


def _want(b, scale):
    return R.attention(b["q"], b["k_cache"], b["v_cache"], b["block_tables"], b["context_lens"], b["cu"],
                       k_scale=b["k_scale"], v_scale=b["v_scale"], scale=scale)


HIDDEN = -240.0  # times any scale below: a weight of 0


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("raised", [False, True])
def test_fp16_results_over_e4m3_stay_at_the_largest_value(raised, new, D, impl):
    """Every V at 65504, and weights that fp16 rounds up: sum P V / sum p passes fp16's largest value by up to 2^-11
    and has to be held there."""
    keys = torch.full((300 + new,), HIDDEN)
    if raised:  # the second key lies 2^7 (1 + 1.02 2^-11) above the first, in another tile: 128 (1 + 2^-10) in fp16
        keys[5], keys[200] = -1.0, 0.0
        scale = math.log(128 * (1 + 1.02 * 2.0 ** -11))
    else:  # 1, and 127 times 0.50026: 0.5 + 2^-11 in fp16
        keys[1:128], keys[0] = -1.0, 0.0
        scale = -math.log(0.50026)
    b = _scored(keys, torch.full_like(keys, 65504.0), new, D, F16, True)
    out, _ = _run(b, scale, impl)
    o, tol, _, _ = _want(b, scale)
    assert abs(float(o.min()) - 65536.0) < 1e-6  # what e4m3 makes of 65504
    R.check(out, o.clamp(max=65504.0), tol + 32)


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("below", [24.6, 25.5])
@pytest.mark.parametrize("sink", [3, 24000])
def test_many_small_weights_beside_a_large_one(sink, below, D, quantised, impl):
    """One key that takes nearly all the weight and holds V = 0 (an attention sink), and the 24576 to 32767 others a
    row sees `below` powers of two under it with V = 1: together they are the result. As many rows as keep a key range
    whole (ranges are joined in fp32).

    In fp16 the weights carry 2^7 and are off by at most half of its smallest step: 2^-25 beside a sum of 2^7 or more,
    2^-32 of each |v|. The other terms are those of ``paged_reference``."""
    n, new, G, bs = 32768, 8192, 4, 16
    g = torch.Generator().manual_seed(62)
    table = torch.randperm(n // bs, generator=g)
    at = table[torch.arange(n) // bs], 0, torch.arange(n) % bs
    k, v = (torch.zeros(n // bs, 1, bs, D, dtype=F16) for _ in range(2))
    k[(*at, 0)] = -1.0
    v[at] = 1.0
    k[table[sink // bs], 0, sink % bs], v[table[sink // bs], 0, sink % bs] = 0.0, 0.0
    ks = vs = None
    if quantised:
        (k, ks), (v, vs) = ((q.float().to(torch.float8_e4m3fn).cuda(), e.float().to(torch.float8_e8m0fnu).cuda())
                            for q, e in (R.quantise(k), R.quantise(v)))
    q = torch.zeros(new, G, D, dtype=F16)
    q[..., 0] = 1
    lse = torch.empty(G, new, device="cuda")
    scale = below * math.log(2)
    out = _paged_attn(q.cuda(), k.cuda(), v.cuda(), table[None].to(torch.int32).cuda(),
                      torch.tensor([n], dtype=torch.int32, device="cuda"),
                      torch.tensor([0, new], dtype=torch.int32, device="cuda"), new, None, 0, ks, vs, scale, None, lse,
                      None, IMPLS[impl])
    others = torch.arange(n - new, n, dtype=torch.float64)  # keys a row sees beside the sink
    w = 2.0 ** -below
    o = others * w / (1 + others * w)
    u, u32 = 2.0 ** -11, 2.0 ** -24
    slack = 2 * (D + 4) * u32 * scale + 2.0 ** -21 + (n + 64) * u32
    tol = (1 + 4 * u) * (2 * u + 2 * slack) * o + 2.0 ** -25 + 2.0 ** -32 * others
    R.check(out, o[:, None, None].expand(out.shape), tol[:, None, None].expand(out.shape))
    l = torch.log1p(others * w)
    R.check(lse, l.expand(lse.shape), (slack + 2.0 ** -22 * (1 + l)).expand(lse.shape), "lse")


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_large_values_in_bf16(new, D, quantised, impl):
    """Values times the keys a row sees (32: two pages are there) just below 2^119, one key 7.9 powers of two above an
    earlier one: its weight may stay at 2^7.9 (a running maximum is raised from 2^8 on)."""
    keys = torch.full((240 + new,), HIDDEN)
    keys[5], keys[192] = -1.0, 0.0
    scale = 7.9 * math.log(2)
    b = _scored(keys, torch.full_like(keys, 1.5 * 2.0 ** 113), new, D, BF16, quantised)
    hidden = torch.ones_like(b["block_tables"], dtype=torch.bool)
    hidden[0, [0, 12]] = False
    b["block_tables"][hidden] = -1
    out, _ = _run(b, scale, impl)
    o, tol, _, _ = _want(b, scale)
    assert 2.0 ** 118 < float(o.max()) * 32 < 2.0 ** 119
    R.check(out, o, tol)
