"""The few-rows paged attention kernel's shared-memory rings: a stage is filled
again, by the copy engine, as soon as its group of keys has been used."""
import re
from pathlib import Path

import pytest
import torch

import paged_reference as R
from lightserve_b200 import _lib
from lightserve_b200.kernels.paged_chunk_attention import _paged_attn

SOURCE = Path(__file__).resolve().parents[1] / "lightserve_b200" / "csrc" / "paged_attn_rows.cu"


def test_a_stage_is_fenced_before_it_is_refilled():
    """In the loop over groups a proxy fence of every lane stands between the last group's reads and the copies
    that go where it was (a vote alone leaves reads that may still be under way)."""
    loop = SOURCE.read_text().split("for (int n = 0; n < mine; ++n) {")[1]
    before = re.sub(r"//[^\n]*", "", loop.split("copy_next(n + AHEAD)")[0])
    fence = before.rfind("fence_async_shared();")
    assert fence >= 0, "the next copies are not ordered behind the reads"
    assert before[:fence].count("{") == before[:fence].count("}"), "the fence must not be conditional"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,quantised", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                             (torch.float16, True)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 2, 4, 6])  # one pair; with 4 heads a group 8, 16 and 24
def test_rings_that_wrap_many_times(new, D, dtype, quantised):
    """Enough CTAs to fill every SM, each ring filled over and over; values of all keys in the result, the same
    bits every time."""
    lens = [2900 - 137 * i for i in range(12)]
    b = R.build(lens, [new] * 12, 4, 4 if new > 1 else 1, D, 16, dtype, quantised=quantised, seed=51)
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}

    def run():
        return _paged_attn(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"], new,
                           None, 0, c["k_scale"], c["v_scale"], None, None, None, None, _lib.IMPL_ROWS)

    out = run()
    o, tol, _, _ = R.attention(b["q"], b["k_cache"], b["v_cache"], b["block_tables"], b["context_lens"], b["cu"],
                               k_scale=b["k_scale"], v_scale=b["v_scale"])
    R.check(out, o, tol)
    assert all(torch.equal(run(), out) for _ in range(30))
