"""Weights and values at the ends of their ranges in attention over a paged cache, by every kernel."""
import math

import pytest
import torch

import paged_reference as R
from lightserve_b200 import _lib
from lightserve_b200.kernels.paged_chunk_attention import _paged_attn

pytestmark = pytest.mark.gpu

F16 = torch.float16
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
