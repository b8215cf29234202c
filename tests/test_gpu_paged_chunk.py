"""Attention of new tokens over a paged cache against the plain 64-bit form:
types, head layouts, page sizes, lengths around every tile edge, windows and
sinks, rows without keys, missing pages, garbage in unused cells, strides,
streams and graphs."""
import pytest
import torch

import paged_reference as R
from lightserve_b200 import _lib
from lightserve_b200.kernels import (flash_attention_varlen, paged_chunk_attention, paged_chunk_workspace,
                                     paged_decode_attention)
from lightserve_b200.kernels.paged_attention import paged_decode_workspace
from lightserve_b200.kernels.paged_chunk_attention import _paged_attn

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _cuda(b):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in b.items()}


def _run(b, window=None, sinks=0, impl=_lib.IMPL_AUTO, most=None, out=None, lse=None, scale=None, workspace=None):
    c = _cuda(b)
    return _paged_attn(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"],
                       b["most"] if most is None else most, window, sinks, c["k_scale"], c["v_scale"], scale,
                       out, lse, workspace, impl)


def _want(b, window=None, sinks=0, most=None, scale=None):
    return R.attention(b["q"], b["k_cache"], b["v_cache"], b["block_tables"], b["context_lens"], b["cu"],
                       window=window, sinks=sinks, k_scale=b["k_scale"], v_scale=b["v_scale"], scale=scale,
                       max_seqlen_q=most)


def _check(b, window=None, sinks=0, impl=_lib.IMPL_AUTO, **kw):
    T, Hq, _ = b["q"].shape
    lse = torch.full((Hq, T), 7.0, device="cuda")
    out = _run(b, window, sinks, impl, lse=lse, **kw)
    o, tol, l, ltol = _want(b, window, sinks, kw.get("most"), kw.get("scale"))
    R.check(out, o, tol)
    R.check(lse, l, ltol, "lse")
    return out, lse


IMPLS = {"auto": _lib.IMPL_AUTO, "simt": _lib.IMPL_SIMT, "rows": _lib.IMPL_ROWS, "tc": _lib.IMPL_TCGEN05}


def _skip_if_not_served(impl, dtype):
    if impl in ("rows", "tc") and dtype == F32:
        pytest.skip("the tensor-core kernels serve 16-bit types")
LENS = [  # cached tokens, new tokens
    ([1], [1]),
    ([40, 17, 1, 0, 16], [3, 17, 1, 0, 16]),            # whole prompts, an empty sequence
    ([15, 16, 17, 31, 32, 33], [1, 2, 3, 4, 5, 6]),
    ([127, 128, 129, 255, 256, 257], [127, 1, 129, 100, 128, 257]),
    ([700, 1030], [300, 5]),
    ([2049, 3], [1, 1]),
]


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("lens,new", LENS)
def test_lengths(lens, new, dtype, D, quantised, impl):
    _skip_if_not_served(impl, dtype)
    _check(R.build(lens, new, 2, 1, D, 16, dtype, quantised=quantised), impl=IMPLS[impl])


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (16, 0), (100, 1), (128, 16), (129, 300), (5000, 4),
                                          (2 ** 40, 2 ** 40)])
@pytest.mark.parametrize("dtype,quantised", [(BF16, False), (F16, True), (F32, False)])
def test_windows(window, sinks, dtype, quantised, impl):
    _skip_if_not_served(impl, dtype)
    b = R.build([9, 300, 1025, 130], [9, 140, 70, 1], 2, 2, 64, 16, dtype, quantised=quantised, seed=3)
    _check(b, window, sinks, IMPLS[impl])


@pytest.mark.parametrize("new", [[1, 1], [140, 9]])
def test_windows_past_every_position(new):
    b = R.build([3000, 77], new, 2, 2, 128, 16, BF16, seed=4)
    plain = _run(b)
    for window, sinks in (((1 << 31) - 1, 0), (1 << 62, 1 << 62), (1 << 70, 1 << 70), (5, 1 << 62)):
        out, _ = _check(b, min(window, 1 << 31), min(sinks, 1 << 31))
        assert torch.equal(_run(b, window, sinks), out)
    assert torch.equal(_run(b, 1 << 62, 1 << 62), plain)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (1, 2), (2, 3), (1, 7), (2, 8), (1, 16), (1, 33)])
@pytest.mark.parametrize("new", [1, 6, 150])
def test_head_groups(H, G, new, quantised):
    _check(R.build([new + 90, new + 40], [new, max(1, new // 2)], H, G, 64, 16, BF16, quantised=quantised, seed=G))


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("bs", [1, 2, 4, 8, 16, 32, 64, 128, 256, 512])
def test_page_sizes(bs, quantised):
    for new in ([1, 1], [200, 33]):
        _check(R.build([600, 333], new, 2, 1, 128, bs, BF16, quantised=quantised, seed=bs))
        _check(R.build([600, 333], new, 2, 1, 128, bs, BF16, quantised=quantised, seed=bs), 70, 3)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [1, 8, 20, 33, 80, 96, 160, 192, 250, 256])
def test_other_head_dims(D, dtype, quantised):
    _check(R.build([70, 40], [20, 1], 2, 2, D, 16, dtype, quantised=quantised, seed=D))


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 9)])
@pytest.mark.parametrize("dtype,D,G,quantised", [(F32, 64, 1, False), (F32, 128, 2, True), (BF16, 96, 1, False),
                                                 (F16, 200, 2, True), (F32, 33, 1, False)])
def test_many_rows_on_the_cuda_cores(dtype, D, G, quantised, window, sinks):
    """Enough query tiles to fill the GPU: 8 pairs a warp."""
    b = R.build([640, 700], [640 // G, 601 // G], 8, G, D, 16, dtype, quantised=quantised, seed=23)
    _check(b, window, sinks, _lib.IMPL_SIMT)


@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [700, 5, 0, 2100]])
@pytest.mark.parametrize("dtype,D,quantised", [(F32, 64, False), (F32, 128, True), (BF16, 96, True), (F16, 250, False),
                                               (F32, 1, False), (BF16, 20, True)])
@pytest.mark.parametrize("window", [None, 40])
def test_one_pair_on_the_cuda_cores(lens, dtype, D, quantised, window):
    """Plain decode there: the warps share one pair."""
    b = R.build(lens, [1] * len(lens), 3, 1, D, 8, dtype, quantised=quantised, seed=24)
    _check(b, window, 2 if window else 0, _lib.IMPL_SIMT)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 20)])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 5], [200, 1, 129]])
def test_missing_pages_hold_no_keys(new, window, sinks, quantised):
    """Ids outside the cache (negative or too large) in the middle, at the start and at the end; a
    sequence whose pages are all missing sees nothing."""
    holes = [(0, 0), (0, 3), (0, 12), (0, 18)] + [(2, i) for i in range(9)]
    b = R.build([300, 60, 140], new, 2, 2, 128, 16, BF16, quantised=quantised, holes=holes, seed=11)
    out, lse = _check(b, window, sinks)
    last = slice(sum(new[:2]), sum(new))
    assert bool((out[last] == 0).all()) and bool((lse[:, last] == float("-inf")).all())


@pytest.mark.parametrize("new", [[12, 5], [300, 200]])
def test_more_rows_than_cached_tokens(new):
    """The first rows stand before position 0 and see nothing."""
    b = R.build([8, 150], new, 2, 1, 64, 16, F16, seed=5)
    out, lse = _check(b)
    assert bool((out[: new[0] - 8] == 0).all()) and bool((lse[:, : new[0] - 8] == float("-inf")).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new", [[3, 2], [140, 20]])
def test_rows_outside_stay(new, dtype):
    """Rows behind the last sequence, and rows past max_seqlen_q, keep what they held."""
    b = R.build([400, 90], new, 2, 1, 128, 16, dtype, seed=6, pad=9)
    most = new[0] - 2
    out = torch.full(b["q"].shape, 3.0, dtype=dtype, device="cuda")
    lse = torch.full((2, b["q"].shape[0]), 5.0, device="cuda")
    _run(b, most=most, out=out, lse=lse)
    o, tol, l, ltol = _want(b, most=most)
    R.check(out, o, tol)
    R.check(lse, l, ltol, "lse")
    rest = o.isnan().any(-1).any(-1)
    assert int(rest.sum()) == 9 + sum(max(0, n - most) for n in new)
    assert bool((out[rest.cuda()] == 3).all()) and bool((lse[:, rest.cuda()] == 5).all())


def test_table_shorter_than_the_context():
    """Keys past the block table's capacity are not read; positions still count them."""
    b = R.build([300, 40], [5, 4], 2, 1, 128, 16, BF16, seed=8)
    b["block_tables"] = b["block_tables"][:, :7].contiguous()
    _check(b)
    _check(b, 250, 3)


@pytest.mark.parametrize("new", [2, 200])
def test_values_before_the_window_do_not_matter(new):
    """Pages that have left every row's window may hold anything, or belong to others."""
    b = R.build([900], [new], 2, 1, 128, 16, BF16, seed=9)
    w, sinks = 100, 5
    gone = b["block_tables"][0, 1:(900 - new - w) // 16].long()
    for c in (b["k_cache"], b["v_cache"]):
        c[gone] = float("nan")
    _check(b, w, sinks)
    b["block_tables"][0, 1:(900 - new - w) // 16] = -1
    _check(b, w, sinks)


def test_nan_in_one_sequence_stays_there():
    b = R.build([64, 64, 300], [1, 64, 200], 1, 1, 128, 16, BF16, seed=10)
    page = int(b["block_tables"][1, 0])
    want = _want(b)
    b["v_cache"][page, :, 0] = float("nan")
    out = _run(b).double().cpu()
    o, tol = want[0].clone(), want[1]
    o[1:65] = float("nan")
    R.check(out, o, tol)
    assert bool(out[1:65].isnan().all())


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [5, 3], [190, 131]])
def test_strided_q_and_out(new, quantised):
    """q as a view of a fused projection, out as a view of a wider buffer, odd offsets included."""
    b = R.build([500, 400], new, 2, 2, 128, 16, BF16, quantised=quantised, seed=12)
    T, H, D = b["q"].shape
    want = _want(b)
    for off in (0, 3, 8):
        wide = torch.zeros(T, 3, H, D + 8 + off, dtype=BF16)
        wide[:, 1, :, off:off + D] = b["q"]
        buf = torch.full((T, H + 1, D + 24), 2.0, dtype=BF16, device="cuda")
        c = _cuda(b)
        q = wide.cuda()[:, 1, :, off:off + D]
        out = buf[:, :H, off:off + D]
        paged_chunk_attention(q, c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"],
                              b["most"], k_scale=c["k_scale"], v_scale=c["v_scale"], out=out)
        R.check(out, want[0], want[1])
        assert bool((buf[:, H] == 2).all()) and bool((buf[:, :, off + D:] == 2).all()) and bool((buf[:, :, :off] == 2).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 12])
def test_unequal_scales(new, D):
    """Quantised rows whose scales span 2^-126 to 2^100: a bf16 cache with rows of zeros and of very small and
    large V beside ordinary ones, and q rows of very different size."""
    b = R.build([200, 300], [new, new], 2, 1, D, 16, BF16, seed=41)
    g = torch.Generator().manual_seed(42)
    shape = b["v_cache"].shape[:3]
    pick = torch.randint(0, 6, shape, generator=g)
    size = torch.tensor([1.0, 1.0, 0.0, 2.0 ** -40, 2.0 ** -110, 2.0 ** 20])[pick][..., None]
    k = torch.randn(*b["k_cache"].shape, generator=g) * torch.exp(torch.randn(*shape, 1, generator=g))
    (kq, ks), (vq, vs) = (R.quantise(x.to(BF16)) for x in (k, torch.randn(*b["v_cache"].shape, generator=g) * size))
    b |= {"k_cache": kq.float().to(torch.float8_e4m3fn), "v_cache": vq.float().to(torch.float8_e4m3fn),
          "k_scale": ks.float().to(torch.float8_e8m0fnu), "v_scale": vs.float().to(torch.float8_e8m0fnu)}
    b["q"] *= torch.exp2(torch.arange(2 * new) * 6.0 - 60).to(BF16)[:, None, None].clamp(max=4)
    _check(b)
    _check(b, impl=_lib.IMPL_SIMT)
    # every V row tiny: the result is as small, not zero
    b["v_scale"].view(torch.uint8).fill_(20)
    _check(b)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("new", [1, 3, 70])
def test_quantised_values_at_the_ends_of_the_range(new, impl, dtype):
    """V rows at fp16's largest value (which e4m3 rounds past it; 2^100 in the types whose sums an fp32
    accumulator must hold) and at the type's smallest: outputs stay finite."""
    _skip_if_not_served(impl, dtype)
    b = R.build([new, 90 + new], [new, new], 2, 1, 64, 16, dtype, seed=43)
    g = torch.Generator().manual_seed(44)
    top, low = 65504.0 if dtype == F16 else 2.0 ** 100, torch.finfo(dtype).smallest_normal / 8
    size = torch.tensor([top, -top, low, 1.0], dtype=torch.float64)
    v = size[torch.randint(0, 4, b["v_cache"].shape[:3], generator=g)][..., None] * torch.ones(64, dtype=torch.float64)
    (kq, ks), (vq, vs) = (R.quantise(x) for x in (torch.randn(*v.shape, generator=g).to(dtype), v.to(dtype)))
    b |= {"k_cache": kq.float().to(torch.float8_e4m3fn), "v_cache": vq.float().to(torch.float8_e4m3fn),
          "k_scale": ks.float().to(torch.float8_e8m0fnu), "v_scale": vs.float().to(torch.float8_e8m0fnu)}
    out = _run(b, impl=IMPLS[impl])
    o, tol, _, _ = _want(b)
    assert bool(out.isfinite().all())
    # fp16's stored value is above its largest, where the result is held
    R.check(out, o.clamp(-top, top), tol + (o.abs() - top).clamp(min=0))


def test_scale_argument():
    b = R.build([200, 60], [70, 1], 2, 1, 64, 16, F16, seed=13)
    for scale in (0.0, 0.5, -0.3):
        _check(b, scale=scale)


def test_large_scores():
    """One key far above the rest, scores near 2^13, and a row of equal scores."""
    b = R.build([513, 140], [200, 1], 1, 1, 128, 16, BF16, seed=14)
    b["q"] *= 16
    b["k_cache"] *= 16
    _check(b)
    b["q"].zero_()
    _check(b)


@pytest.mark.parametrize("dtype,quantised", [(BF16, False), (BF16, True), (F32, False)])
def test_decode_form_is_one_row_per_sequence(dtype, quantised):
    lens = [1, 16, 700, 0, 2100, 33]
    b = R.build(lens, [1] * 6, 2, 2, 128, 16, dtype, quantised=quantised, seed=15)
    c = _cuda(b)
    for window, sinks in ((None, 0), (64, 4), (700, 0)):
        o, tol, _, _ = R.attention(b["q"], b["k_cache"], b["v_cache"], b["block_tables"], b["context_lens"], None,
                                   window=window, sinks=sinks, k_scale=b["k_scale"], v_scale=b["v_scale"])
        ws = paged_decode_workspace(b["q"].shape, b["block_tables"].shape[1], 16, "cuda", num_kv_heads=2,
                                    quantized=quantised, window=window, num_sinks=sinks)
        out = paged_decode_attention(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"],
                                     window=window, num_sinks=sinks, k_scale=c["k_scale"], v_scale=c["v_scale"],
                                     workspace=ws)
        R.check(out, o, tol)
        assert bool((out[3] == 0).all())


def test_plain_decode_call_is_unchanged():
    """Without the new arguments the decode call takes the kernel it always took: bit-identical to its C entry."""
    b = R.build([1, 513, 1500], [1] * 3, 4, 1, 128, 16, BF16, seed=16)
    c = _cuda(b)
    out = paged_decode_attention(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"])
    lib, ref = _lib.load(), torch.empty_like(c["q"])
    S, H, D = b["q"].shape
    nb, _, bs, _ = b["k_cache"].shape
    mb = b["block_tables"].shape[1]
    need = lib.lsb_paged_decode_workspace_size(S, H, D, mb, bs)
    ws = torch.empty(need // 4 + 1, device="cuda")
    _lib.check(lib.lsb_paged_decode(
        c["q"].data_ptr(), c["k_cache"].data_ptr(), c["v_cache"].data_ptr(), c["block_tables"].data_ptr(),
        c["context_lens"].data_ptr(), ref.data_ptr(), S, H, D, mb, bs, nb, H * D, D, H * D, D, 1 / D ** 0.5,
        _lib.DTYPE_BF16, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "lsb_paged_decode")
    assert torch.equal(out, ref)


def test_whole_prompts_match_packed_prefill():
    """With nothing cached before the chunk the operator is the packed causal prefill."""
    lens = [300, 1, 129]
    b = R.build(lens, lens, 2, 1, 128, 16, BF16, seed=17)
    c = _cuda(b)
    rows = torch.cat([torch.arange(n) for n in lens])
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])
    ids = b["block_tables"][seq, rows // 16].long()
    k, v = (b[n][ids, :, rows % 16].cuda() for n in ("k_cache", "v_cache"))
    ref = flash_attention_varlen(c["q"], k, v, c["cu"], max(lens), causal=True)
    out = _run(b)
    o, tol, _, _ = _want(b)
    R.check(out, o, tol)
    R.check(ref, o, tol)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 3, 2], [150, 1, 260]])
@pytest.mark.parametrize("D,G", [(128, 2), (64, 8)])
def test_same_inputs_same_bits(D, G, new, quantised):
    b = R.build([1500, 64, 800], new, 2, G, D, 16, BF16, quantised=quantised, seed=18)
    c = _cuda(b)
    outs = [paged_chunk_attention(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"],
                                  b["most"], window=400, num_sinks=4, k_scale=c["k_scale"], v_scale=c["v_scale"])
            for _ in range(20)]
    assert all(torch.equal(outs[0], o) for o in outs)


def test_two_calls_on_two_streams():
    b = [R.build([900, 77], [5 + 60 * i, 20], 2, 1, 128, 16, BF16, seed=19 + i, quantised=bool(i)) for i in range(2)]
    c = [_cuda(x) for x in b]
    streams = [torch.cuda.Stream() for _ in b]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for x, st in zip(c, streams):
            with torch.cuda.stream(st):
                outs.append(paged_chunk_attention(x["q"], x["k_cache"], x["v_cache"], x["block_tables"],
                                                  x["context_lens"], x["cu"], x["most"], k_scale=x["k_scale"],
                                                  v_scale=x["v_scale"]))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        o, tol, _, _ = _want(b[i % 2])
        R.check(out, o, tol)


@pytest.mark.parametrize("quantised", [False, True])
def test_captured_graph_follows_its_buffers(quantised):
    """Two captured graphs with workspaces of their own, replayed in turn with an eager call between, see the
    lengths and tables as they are at each replay."""
    graphs = []
    for i, new in enumerate(([1, 1, 1], [130, 3, 1])):
        b = R.build([900, 40, 300], new, 2, 2, 128, 16, BF16, quantised=quantised, seed=30 + i)
        c = _cuda(b)
        out = torch.empty_like(c["q"])
        ws = paged_chunk_workspace(c["q"].shape, 3, b["most"], 2, c["block_tables"].shape[1], 16, "cuda", 256, 4)

        def call(c=c, out=out, ws=ws, most=b["most"]):
            paged_chunk_attention(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"],
                                  most, window=256, num_sinks=4, k_scale=c["k_scale"], v_scale=c["v_scale"],
                                  out=out, workspace=ws)

        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append((b, c, out, g))
    for lens in ([900, 40, 300], [131, 39, 7], [800, 3, 16]):
        for b, c, out, g in graphs:
            b["context_lens"] = torch.tensor(lens, dtype=torch.int32)
            c["context_lens"].copy_(b["context_lens"])
            out.fill_(9)
            g.replay()
            _run(graphs[0][0])
        torch.cuda.synchronize()
        for b, c, out, g in graphs:
            o, tol, _, _ = _want(b, 256, 4)
            R.check(out, o, tol)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("new", [1, 3, 140])
def test_offsets_past_32_bits(new, quantised):
    """Pages at the far end of a cache of more than 2^31 elements."""
    H, bs, D = 16, 16, 128
    nb = 2 ** 31 // (H * bs * D) + 40
    b = R.build([333], [new], H, 1, D, bs, BF16, quantised=quantised, seed=21)
    c = _cuda(b)
    far = {}
    for n in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if b[n] is None:
            far[n] = None
            continue
        small = c[n].view(torch.uint8) if quantised else c[n]
        big = torch.empty(nb, *small.shape[1:], dtype=small.dtype, device="cuda")
        big[-small.shape[0]:] = small
        far[n] = big.view(c[n].dtype)
    shift = nb - b["k_cache"].shape[0]
    bt = torch.where(c["block_tables"] >= 0, c["block_tables"] + shift, c["block_tables"]).to(torch.int32)
    out = paged_chunk_attention(c["q"], far["k_cache"], far["v_cache"], bt, c["context_lens"], c["cu"], new,
                                k_scale=far["k_scale"], v_scale=far["v_scale"])
    o, tol, _, _ = _want(b)
    R.check(out, o, tol)


def test_empty_calls():
    b = R.build([5, 6], [0, 0], 2, 1, 64, 16, BF16, pad=3)
    c = _cuda(b)
    out = torch.full_like(c["q"], 4)
    for most in (0, 2):
        paged_chunk_attention(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"], c["cu"], most,
                              out=out)
    none = paged_chunk_attention(c["q"][:0], c["k_cache"], c["v_cache"], c["block_tables"][:0].contiguous(),
                                 c["context_lens"][:0], c["cu"][:1], 0)
    assert bool((out == 4).all()) and none.shape == (0, 2, 64)
