"""The paged-cache operators together, as the decoder and the serving engine run
them: prompts prefilled in chunks over the cache, a sliding window with sinks, an
e4m3 cache, decode steps in a CUDA graph. Tokens are compared with a plain
full-recompute forward that applies the same window and stores K/V through the
64-bit form of the quantisation."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import paged_reference as R
from conftest import GOLDEN
from oracle.llama import _rope_tables, _rot
from lightserve_b200.engine import BlockManager, CacheConfig, Request, SamplingParams, SchedulerConfig
from lightserve_b200.model.minimal_llama import LlamaConfig, init_weights
from lightserve_b200.model.paged_decode import PagedDecoder, PagedKVCache
from lightserve_b200.model.serving import ServingEngine

pytestmark = pytest.mark.gpu

PROMPTS = (37, 5, 16, 1)


def _toy(dtype, max_seq_len=128):
    return LlamaConfig(vocab_size=256, hidden_size=256, intermediate_size=688, n_layers=2, n_heads=4, head_dim=64,
                       max_seq_len=max_seq_len, rope_theta=10000.0, dtype=dtype)


def _decoder(cfg, n, quantized=False, **options):
    cache = PagedKVCache(cfg, num_blocks=64, block_size=16, quantized=quantized)
    bm = BlockManager(block_size=16, num_gpu_blocks=64)
    return PagedDecoder(init_weights(cfg, device="cuda", seed=0), cfg, cache, bm, max_batch=n, max_blocks_per_seq=8,
                        **options)


def _prompts(lens=PROMPTS, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (n,), generator=g).tolist() for n in lens]


def _logits(w, cfg, ids, window=None, sinks=0, quantized=False):
    """Logits of the last position of one sequence (fp32 CPU weights)."""
    N = len(ids)
    cos, sin = (t[:N, None] for t in _rope_tables(cfg))
    keep = R.visible(torch.arange(N), N, window, sinks)

    def norm(h, g):
        return h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + cfg.rms_eps) * g

    def stored(x):
        q, e = R.quantise(x)
        return (q * e[..., None]).float()

    r = F.embedding(torch.tensor(ids), w.embed_tokens)
    for layer in w.layers:
        h = norm(r, layer.input_layernorm_weight)
        q, k, v = ((h @ m).view(N, cfg.n_heads, cfg.head_dim) for m in (layer.q_proj, layer.k_proj, layer.v_proj))
        q, k = q * cos + _rot(q) * sin, k * cos + _rot(k) * sin
        if quantized:
            k, v = stored(k), stored(v)
        s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(cfg.head_dim)
        a = torch.softmax(s.masked_fill(~keep, -math.inf), -1)
        r = r + torch.einsum("hij,jhd->ihd", a, v).reshape(N, -1) @ layer.o_proj
        h = norm(r, layer.post_attention_layernorm_weight)
        r = r + (F.silu(h @ layer.gate_proj) * (h @ layer.up_proj)) @ layer.down_proj
    return norm(r, w.norm_weight)[-1] @ w.lm_head


@pytest.mark.parametrize("chunk", [1, 7, 16, 1000])
def test_fp32_chunked_prefill_gives_the_reference_tokens(chunk):
    """fp32, no window, plain cache: exactly lightserve's full-recompute greedy tokens, whatever the chunk size."""
    g = np.load(GOLDEN / "llama_toy.npz")
    prompts = [list(map(int, row[:n])) for row, n in zip(g["prompts"], g["prompt_lens"])]
    steps = g["tokens"].shape[1]
    dec = _decoder(_toy(torch.float32, 64), len(prompts), prefill_chunk_tokens=chunk)
    out = dec.generate([Request(f"r{i}", p, SamplingParams(max_tokens=steps)) for i, p in enumerate(prompts)], steps)
    assert out == [list(map(int, t)) for t in g["tokens"]]


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("quantized,window,sinks,chunk", [(True, None, 0, None), (False, 12, 3, None), (True, 12, 3, 11),
                                                          (True, None, 0, 20), (False, 40, 0, 16)])
def test_tokens_match_a_plain_forward(quantized, window, sinks, chunk, dtype, use_graph):
    """Each token is the argmax of the plain forward on the same prefix, wherever that forward's top-2 margin
    exceeds the noise: fp32 1e-3 (a K/V value next to a rounding border of e4m3 may fall on the other side: up to 2^-3
    of that element), bf16 0.05 as in the other decode tests."""
    cfg = _toy(dtype)
    dec = _decoder(cfg, len(PROMPTS), quantized, window=window, num_sinks=sinks, prefill_chunk_tokens=chunk)
    prompts, steps = _prompts(), 9
    out = dec.generate([Request(f"r{i}", p) for i, p in enumerate(prompts)], steps, use_graph=use_graph)
    w = init_weights(_toy(torch.float32), device="cpu", seed=0)
    checked, total = 0, 0
    for p, toks in zip(prompts, out):
        ids = list(p)
        for t in toks:
            top = torch.topk(_logits(w, _toy(torch.float32), ids, window, sinks, quantized), 2)
            total += 1
            if float(top.values[0] - top.values[1]) > (1e-3 if dtype == torch.float32 and not quantized else
                                                       0.02 if dtype == torch.float32 else 0.05):
                assert t == int(top.indices[0])
                checked += 1
            ids.append(t)  # teacher-force our own token
    assert checked >= total // 2


def test_bf16_chunks_fill_the_cache_like_the_packed_prefill():
    """First-layer K/V depend on the tokens alone: equal bit for bit however the prompt is cut."""
    cfg = _toy(torch.bfloat16)
    caches = []
    for chunk in (None, 13):
        dec = _decoder(cfg, len(PROMPTS), prefill_chunk_tokens=chunk)
        dec.admit([Request(f"r{i}", p) for i, p in enumerate(_prompts())], 2)
        caches.append((dec.cache.k, dec.cache.v))
    for a, b in zip(*caches):
        assert torch.equal(a[0], b[0])
        torch.testing.assert_close(a[1].float(), b[1].float(), atol=3e-2, rtol=3e-2)


def test_quantized_cache_is_the_quantised_plain_cache():
    """First-layer rows of an e4m3 decoder are the quantised rows of a bf16 one, after prefill and decode steps."""
    from lightserve_b200.kernels import dequantize_kv_cache

    cfg = _toy(torch.bfloat16)
    a, b = (_decoder(cfg, len(PROMPTS), q, prefill_chunk_tokens=9) for q in (False, True))
    for d in (a, b):
        d.admit([Request(f"r{i}", p) for i, p in enumerate(_prompts())], 4)
    b.tokens.copy_(a.tokens)
    a.step(), b.step()
    assert torch.equal(a.context_lens, b.context_lens)
    slots = torch.cat([torch.tensor([t for t in row.tolist() if t >= 0])[: -(-int(c) // 16)].repeat_interleave(16)[: int(c)] * 16
                       + torch.arange(int(c)) % 16 for row, c in zip(a.block_tables, a.context_lens)]).cuda()
    k, v = dequantize_kv_cache(b.cache.k[0], b.cache.v[0], b.cache.k_scale[0], b.cache.v_scale[0], slots, torch.bfloat16)
    for got, pool in ((k, a.cache.k[0]), (v, a.cache.v[0])):
        q, e = R.quantise(pool[slots // 16, :, slots % 16].cpu())
        assert torch.equal(got.double().cpu(), q * e[..., None])


@pytest.mark.parametrize("options", [{"prefill_chunk_tokens": 6}, {"quantized_kv": True},
                                     {"window": 10, "num_sinks": 2, "quantized_kv": True, "prefill_chunk_tokens": 16}])
@pytest.mark.parametrize("blocks", [64, 16])  # 16: the three running requests outgrow the pool
def test_serving_with_options(options, blocks):
    """Through the scheduler, with requests queueing and being recomputed, every option gives the tokens that the
    same decoder gives without a scheduler."""
    cfg = _toy(torch.float32)
    prompts, steps = _prompts((30, 9, 17, 2), 8), 8
    eng = ServingEngine(init_weights(cfg, device="cuda", seed=0), cfg, CacheConfig(block_size=4, num_gpu_blocks=blocks),
                        SchedulerConfig(max_num_seqs=3, max_num_batched_tokens=256), **options)
    out = eng.generate(prompts, max_tokens=steps)
    o = dict(options)
    dec = _decoder(cfg, len(prompts), o.pop("quantized_kv", False), **o)
    ref = dec.generate([Request(f"r{i}", p) for i, p in enumerate(prompts)], steps)
    w = init_weights(cfg, device="cpu", seed=0)
    for p, got, want in zip(prompts, out, ref):
        for i, (a, b) in enumerate(zip(got, want)):
            if a != b:  # only where two orders of the same sums may part
                top = torch.topk(_logits(w, cfg, p + want[:i], o.get("window"), o.get("num_sinks", 0),
                                         options.get("quantized_kv", False)), 2).values
                assert float(top[0] - top[1]) < 0.02
                break
    if blocks == 16:
        assert eng.num_preemptions > 0


def test_cache_sizes():
    cfg = _toy(torch.bfloat16)
    plain, small = (PagedKVCache(cfg, 8, 16, quantized=q).nbytes() for q in (False, True))
    assert plain == 2 * 2 * 8 * 4 * 16 * 64 * 2 and small == 2 * 2 * 8 * 4 * 16 * (64 + 1)


def test_prefill_over_the_cache_only():
    dec = _decoder(_toy(torch.bfloat16), 1, True)
    with pytest.raises(AssertionError, match="over the cache"):
        dec.admit([Request("r", [1, 2])], 2, packed=False)
    with pytest.raises(AssertionError, match="positive"):
        _decoder(_toy(torch.bfloat16), 1, prefill_chunk_tokens=0)
    with pytest.raises(AssertionError, match="needs a window"):
        _decoder(_toy(torch.bfloat16), 1, num_sinks=2)
