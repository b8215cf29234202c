"""The paged-cache operators of serving beyond the one-shot prefill, as cases to be timed and compared.

Four kinds of case, one for each way the operators are called:

* ``chunk``:  attention of a chunk of new tokens over a paged cache (the K/V of the chunk already in it), over a
  16-bit, 32-bit or e4m3 cache, optionally with a sliding window and a few first tokens that stay visible;
* ``decode``: the same for one new token per sequence;
* ``store``:  K/V rows quantised to e4m3 as they are written into the cache, and read back from it;
* ``rope``:   rotary embedding, quantisation and cache write of a fused QKV projection in one call (a prompt's
  tokens by cache slot, or a decode step's by block table), the rows read back likewise.

``run`` computes either their plain form from elementary torch operations, or (``own``) makes the calls of this
package. A quantised row is 8-bit e4m3 values with one power-of-two scale (e8m0) for each token and head.
"""
import math
import random

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _attend(name, kind, dtype, cache, seqs, new, ctx, heads, group, dim, block=16, window=0, sinks=0, spread=1):
    """seqs sequences of ctx[0]..ctx[1] cached tokens, new[0]..new[1] of which are the chunk's; heads counts the
    cache's heads and group the query heads that share one; window 0 is none."""
    c = {"kind": kind, "dtype": dtype, "cache": cache, "seqs": seqs, "new_min": new[0], "new_max": new[1],
         "ctx_min": ctx[0], "ctx_max": ctx[1], "heads": heads, "group": group, "dim": dim, "block": block,
         "window": window, "sinks": sinks, "spread": spread}
    return dict(c, name=name) if name else c


def _rows(name, kind, dtype, tokens, heads, dim, block=16, step=False):
    c = {"kind": kind, "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim, "block": block, "step": step}
    return dict(c, name=name) if name else c


def listed():
    return [
        # The last 2048 tokens of an 8192-token prompt, prefilled in chunks, at the decode benchmark's heads.
        _attend("chunk prompt", "chunk", "bf16", "same", 1, (2048, 2048), (8192, 8192), 16, 1, 128),
        # Eight prompts prefilled side by side in a chunk budget of 4096 tokens over a quantised cache.
        _attend("chunk batch e4m3", "chunk", "bf16", "e4m3", 8, (300, 724), (724, 4096), 16, 1, 128, spread=2),
        # Long conversations that keep 1024 tokens and the first four: a chunk each.
        _attend("chunk window", "chunk", "fp16", "same", 4, (700, 1031), (2000, 16383), 8, 4, 64, window=1024, sinks=4),
        # Drafted tokens of 32 sequences verified in one pass: one to five rows each.
        _attend("chunk drafts", "chunk", "bf16", "same", 32, (1, 5), (512, 4096), 8, 4, 128, spread=3),
        # The fp32 toy decoder of the tests: the smallest call, where latency counts.
        _attend("chunk toy fp32", "chunk", "fp32", "same", 3, (5, 33), (33, 64), 4, 1, 64),
        # The decode benchmark's 64 sequences over a quantised cache.
        _attend("decode e4m3", "decode", "bf16", "e4m3", 64, (1, 1), (512, 4096), 16, 1, 128, spread=4),
        # One user, one long conversation, shared heads.
        _attend("decode one e4m3", "decode", "fp16", "e4m3", 1, (1, 1), (30011, 30011), 8, 4, 64),
        # 48 long sequences that keep a window and the first tokens.
        _attend("decode window", "decode", "bf16", "same", 48, (1, 1), (900, 12000), 16, 1, 128, window=2048, sinks=16),
        # A packed prefill's K/V (16384 tokens), and a decode step's.
        _rows("store prompt", "store", "bf16", 16384, 16, 128),
        _rows("store step", "store", "fp16", 64, 16, 64),
        _rows("rope prompt", "rope", "bf16", 12001, 16, 128),
        _rows("rope step", "rope", "bf16", 64, 16, 128, step=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "decode", "decode", "store", "rope"])
    if kind in ("store", "rope"):
        dim, heads = rng.choice([64, 128]), rng.choice([1, 4, 8, 16, 32])
        step = kind == "rope" and rng.random() < 0.5
        tokens = _log(rng, 1, 256) if step else _log(rng, 1, 32_000_000 // (heads * dim))
        return _rows("", kind, rng.choice(["bf16", "fp16", "fp32"]), tokens, heads, dim, rng.choice([8, 16, 32]), step)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    cache = rng.choice(["same", "e4m3"])
    heads, group, dim = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([64, 128])
    seqs = _log(rng, 1, 64)
    new = _log(rng, 1, 2048) if kind == "chunk" else 1
    # Cached tokens, so that no case costs more than the largest listed one: the read of the cache is held to
    # 300 MB, the products to 40 GFLOP (fp32: 2 GFLOP).
    most = min(32768, 300_000_000 // (seqs * heads * dim * 8),
               (2_000_000_000 if dtype == "fp32" else 40_000_000_000) // (4 * seqs * new * heads * group * dim))
    new = max(1, min(new, most))
    hi = max(new, _log(rng, max(1, min(64, most)), max(2, most)))
    lo = max(1, hi // rng.choice([1, 2, 8]))
    window = _log(rng, 1, 4096) if rng.random() < 0.4 else 0
    return _attend("", kind, dtype, cache, seqs, (max(1, new // rng.choice([1, 3])), new), (lo, hi), heads, group, dim,
                   rng.choice([8, 16, 16, 32]), window, rng.choice([0, 1, 4, 37]) if window else 0,
                   spread=rng.randrange(1 << 20))


def _lens(case):
    """(new, cached) tokens of each sequence; the cached ones include the new ones."""
    r = random.Random(case["spread"])
    ctx = [r.randint(case["ctx_min"], case["ctx_max"]) for _ in range(case["seqs"])]
    return [(min(r.randint(case["new_min"], case["new_max"]), c), c) for c in ctx]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _kv(g, *shape):
    """K or V values as a model makes them: some channels and some tokens are larger than others."""
    x = _normal(g, *shape) * torch.exp(0.3 * _normal(g, *shape[:-1], 1))
    return x * torch.exp(0.3 * _normal(g, *([1] * (len(shape) - 1)), shape[-1]))


def _quantise(x):
    """x (fp32) as e4m3 values and a power-of-two scale for each row: the smallest that takes the row's largest
    magnitude to 448 or less. NaN and infinities become NaN and leave the scale alone."""
    finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    m, e = torch.frexp(finite.amax(-1))                # largest = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.clamp(e - 9 + (m > 0.875), min=-126)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    q = torch.ldexp(x, -e.unsqueeze(-1))
    return q.to(torch.float8_e4m3fn), torch.ldexp(torch.ones_like(m), e).to(torch.float8_e8m0fnu)


def _prepare_attend(case, g):
    lens = _lens(case)
    heads, group, dim, block, dtype = case["heads"], case["group"], case["dim"], case["block"], TYPES[case["dtype"]]
    per = max(-(-c // block) for _, c in lens)
    pages = sum(-(-c // block) for _, c in lens) + 3
    ids = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((case["seqs"], per), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for s, (_, c) in enumerate(lens):
        n = -(-c // block)
        table[s, :n] = ids[at:at + n]
        at += n
    cu = [0]
    for n, _ in lens:
        cu.append(cu[-1] + n)
    s = {"kind": case["kind"], "q": _normal(g, cu[-1], heads * group, dim).to(dtype), "table": table,
         "ctx": torch.tensor([c for _, c in lens], dtype=torch.int32, device=DEVICE),
         "cu": torch.tensor(cu, dtype=torch.int32, device=DEVICE), "most": max(n for n, _ in lens),
         "window": case["window"] or None, "sinks": case["sinks"], "k_scale": None, "v_scale": None}
    k, v = _kv(g, pages, heads, block, dim), _kv(g, pages, heads, block, dim)
    if case["cache"] == "e4m3":
        s["k"], s["k_scale"] = _quantise(k.to(dtype).float())
        s["v"], s["v_scale"] = _quantise(v.to(dtype).float())
    else:
        s["k"], s["v"] = k.to(dtype), v.to(dtype)
    return s


def _prepare_rows(case, g):
    tokens, heads, dim, block, dtype = case["tokens"], case["heads"], case["dim"], case["block"], TYPES[case["dtype"]]
    pages = -(-tokens // block) + 3
    s = {"kind": case["kind"], "dtype": dtype, "step": case["step"], "block": block}
    for n in ("k", "v"):
        s[n + "_cache"] = torch.zeros(pages, heads, block, dim, device=DEVICE).to(torch.float8_e4m3fn)
        s[n + "_scale"] = torch.zeros(pages, heads, block, dtype=torch.uint8, device=DEVICE).view(torch.float8_e8m0fnu)
    s["slots"] = torch.randperm(pages * block, generator=g, device=DEVICE)[:tokens].contiguous()
    if case["kind"] == "store":
        s["k"], s["v"] = (_kv(g, tokens, heads, dim).to(dtype) for _ in range(2))
        return s
    s["qkv"] = _kv(g, tokens, 3, heads, dim).to(dtype)
    far = 4096
    angle = torch.outer(torch.arange(far, device=DEVICE, dtype=torch.float64),
                        500000.0 ** -(torch.arange(dim // 2, device=DEVICE, dtype=torch.float64) / (dim // 2)))
    s["cos"], s["sin"] = (torch.cat([t, t], -1).to(dtype).contiguous() for t in (angle.cos(), angle.sin()))
    s["q_out"] = torch.empty(tokens, heads, dim, dtype=dtype, device=DEVICE)
    s["positions"] = torch.randint(far, (tokens,), generator=g, device=DEVICE)
    if case["step"]:  # one token of each of `tokens` sequences, each writing to a page of its own
        pages = tokens + 3
        for n in ("k", "v"):
            s[n + "_cache"] = torch.zeros(pages, heads, block, dim, device=DEVICE).to(torch.float8_e4m3fn)
            s[n + "_scale"] = torch.zeros(pages, heads, block, dtype=torch.uint8, device=DEVICE).view(torch.float8_e8m0fnu)
        page = torch.randperm(pages, generator=g, device=DEVICE)[:tokens]
        s["table"] = torch.full((tokens, far // block), -1, dtype=torch.int32, device=DEVICE)
        s["table"][torch.arange(tokens, device=DEVICE), s["positions"] // block] = page.to(torch.int32)
        s["ctx"] = torch.zeros(tokens, dtype=torch.int32, device=DEVICE)
        s["slots"] = page * block + s["positions"] % block
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return (_prepare_attend if case["kind"] in ("chunk", "decode") else _prepare_rows)(case, g)


def _pages(cache, scale, table):
    """The cached rows of each sequence in fp32, [seqs, heads, 1, tokens, dim]."""
    at = table.clamp(min=0).long()
    x = cache[at].float()
    if scale is not None:
        x = x * scale[at].float().unsqueeze(-1)
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).unsqueeze(2)


def _plain_attend(s):
    q, cu, ctx, heads = s["q"], s["cu"].long(), s["ctx"].long(), s["k"].shape[1]
    tokens, dim = q.shape[0], q.shape[2]
    # The chunk's rows as a padded batch: row i of sequence b is token cu[b] + i.
    i = torch.arange(s["most"], device=q.device)
    row = (cu[:-1, None] + i).clamp(max=tokens - 1)
    x = q[row].float().unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4)           # [seqs, heads, group, rows, dim]
    x = x @ _pages(s["k"], s["k_scale"], s["table"]).transpose(-1, -2)
    x = x * (1.0 / math.sqrt(dim))
    place = (ctx - (cu[1:] - cu[:-1]))[:, None, None] + i[None, :, None]          # each row's position
    key = torch.arange(x.shape[-1], device=q.device)
    seen = (key <= place) & (key < ctx[:, None, None])
    if s["window"] is not None:
        seen = seen & ((place - key < s["window"]) | (key < s["sinks"]))
    x = torch.where(seen[:, None, None], x, torch.full_like(x, -math.inf))
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = x.sum(-1, keepdim=True)
    x = (x @ _pages(s["v"], s["v_scale"], s["table"])) / torch.where(total > 0, total, torch.ones_like(total))
    t = torch.arange(tokens, device=q.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    return x.permute(0, 3, 1, 2, 4).flatten(2, 3)[b, t - cu[b]].to(q.dtype)


def _plain_rope(x, cos, sin):
    """The model's rotary embedding: rotate-half, each product and the sum rounded to the model's type, which
    the cached values are defined by."""
    half, t = x.shape[-1] // 2, x.dtype
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    a, b = (x.float() * cos.float()).to(t), (turned.float() * sin.float()).to(t)
    return (a.float() + b.float()).to(t)


def _plain_stored(x, dtype):
    """What e4m3 storage makes of rows x, as values of the model's type."""
    q, e = _quantise(x.float())
    most = torch.finfo(dtype).max
    return (q.float() * e.float().unsqueeze(-1)).clamp(-most, most).to(dtype)


def _plain(s):
    if s["kind"] in ("chunk", "decode"):
        return _plain_attend(s)
    if s["kind"] == "store":
        return {"k": _plain_stored(s["k"], s["dtype"]), "v": _plain_stored(s["v"], s["dtype"])}
    cos, sin = s["cos"][s["positions"], None], s["sin"][s["positions"], None]
    return {"q": _plain_rope(s["qkv"][:, 0], cos, sin),
            "k": _plain_stored(_plain_rope(s["qkv"][:, 1], cos, sin), s["dtype"]),
            "v": _plain_stored(s["qkv"][:, 2], s["dtype"])}


def _own(s):
    from lightserve_b200 import kernels as K

    quantised = [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if n in s]
    if s["kind"] == "chunk":
        return K.paged_chunk_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], s["most"],
                                       window=s["window"], num_sinks=s["sinks"], k_scale=s["k_scale"],
                                       v_scale=s["v_scale"])
    if s["kind"] == "decode":
        return K.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], window=s["window"],
                                        num_sinks=s["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["kind"] == "store":
        K.quantize_kv_cache(s["k"], s["v"], *quantised, s["slots"])
        k, v = K.dequantize_kv_cache(*quantised, s["slots"], s["dtype"])
        return {"k": k, "v": v}
    if s["step"]:
        K.rope_quantize_kv(s["qkv"], s["cos"], s["sin"], s["positions"], s["q_out"], *quantised,
                           block_tables=s["table"], context_lens=s["ctx"])
    else:
        K.rope_quantize_kv(s["qkv"], s["cos"], s["sin"], s["positions"], s["q_out"], *quantised,
                           slot_mapping=s["slots"])
    k, v = K.dequantize_kv_cache(*quantised, s["slots"], s["dtype"])
    return {"q": s["q_out"], "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    heads, dim = case["heads"], case["dim"]
    if case["kind"] in ("store", "rope"):
        row = case["tokens"] * heads * dim
        cell = 2 * (row + case["tokens"] * heads)                   # e4m3 rows of K and V and their scales
        read = row * SIZE[case["dtype"]] * (2 if case["kind"] == "store" else 3)
        more = 0 if case["kind"] == "store" else row * SIZE[case["dtype"]] + 2 * case["tokens"] * dim * SIZE[case["dtype"]]
        return {"bytes": read + more + 2 * cell + 2 * row * SIZE[case["dtype"]], "flops": 4 * row}
    window = case["window"] or 1 << 40
    kept, pairs, rows = 0, 0, 0
    for n, c in _lens(case):
        first = max(0, c - n - window + 1)                          # the first key in any row's window
        kept += c - first + min(first, case["sinks"])
        pairs += sum(min(p + 1, window + min(case["sinks"], max(0, p + 1 - window))) for p in range(c - n, c))
        rows += n
    cell = dim + 1 if case["cache"] == "e4m3" else dim * SIZE[case["dtype"]]
    lanes = heads * case["group"] * dim
    return {"bytes": 2 * kept * heads * cell + 2 * rows * lanes * SIZE[case["dtype"]], "flops": 4 * pairs * lanes}


def exact(case, seed):
    s = prepare(case, seed)
    wide = torch.float64

    def stored(x):  # by hand: 3 mantissa bits down to 2^-6, steps of 2^-9 below it
        x = x.to(wide)
        top = x.abs().amax(-1, keepdim=True)
        up = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / 448)).clamp(min=-126)
        up = torch.where(top > 448 * torch.exp2(up), up + 1, up)
        up = torch.where((top <= 448 * torch.exp2(up - 1)) & (up > -126), up - 1, up)
        y = x * torch.exp2(-up)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        most = torch.finfo(s["dtype"]).max
        return (torch.round(y / step) * step * torch.exp2(up)).clamp(-most, most)

    if case["kind"] == "store":
        return {"k": stored(s["k"]), "v": stored(s["v"])}
    if case["kind"] == "rope":
        half, t = case["dim"] // 2, s["dtype"]
        cos, sin = s["cos"].to(wide)[s["positions"], None], s["sin"].to(wide)[s["positions"], None]

        def turn(x):
            x1, x2, short = x[..., :half].to(wide), x[..., half:].to(wide), lambda y: y.to(t).to(wide)
            return short(torch.cat([short(x1 * cos[..., :half]) - short(x2 * sin[..., :half]),
                                    short(x2 * cos[..., half:]) + short(x1 * sin[..., half:])], -1))

        return {"q": turn(s["qkv"][:, 0]), "k": stored(turn(s["qkv"][:, 1])), "v": stored(s["qkv"][:, 2])}
    heads, group, dim = case["heads"], case["group"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=wide, device=DEVICE)
    at = 0
    for b, (n, c) in enumerate(_lens(case)):
        ids = s["table"][b, :-(-c // case["block"])].long()
        k, v = s["k"][ids].to(wide), s["v"][ids].to(wide)           # [pages, heads, block, dim]
        if case["cache"] == "e4m3":
            k, v = k * s["k_scale"][ids].to(wide)[..., None], v * s["v_scale"][ids].to(wide)[..., None]
        for h in range(heads):
            kh, vh = k[:, h].reshape(-1, dim)[:c], v[:, h].reshape(-1, dim)[:c]
            p = torch.arange(c - n, c, device=DEVICE)[:, None]
            j = torch.arange(c, device=DEVICE)[None]
            hidden = j > p
            if case["window"]:
                hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
            x = s["q"][at:at + n, h * group:(h + 1) * group].to(wide).transpose(0, 1) @ kh.T / dim ** 0.5
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h * group:(h + 1) * group] = (x @ vh).transpose(0, 1)
        at += n
    return out
