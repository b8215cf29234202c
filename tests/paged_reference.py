"""Plain 64-bit forms of the paged-cache operators (CPU), with error bounds.

Bounds (``attention``): o = sum_j p_j v_j / sum_j p_j. Write A = sum_j p_j |v_j| /
sum_j p_j, N for the keys and D for the head dim, u = eps(dtype) / 2 for one
rounding to the output type, u32 = 2^-24.
* A score is a dot product of D products summed in fp32 and scaled twice:
  off by at most ds = (D + 4) u32 scale sum_d |q_d k_jd|; exp2 adds its argument's
  rounding (within ds again, |score| <= scale sum |q k|) and 2^-21 for the function.
  So p_j is off by a factor 1 +- g, g = 2 ds + 2^-21, numerator and denominator
  each, 2 g A together.
* Sums of N terms in fp32, the rescaling and the joining of split ranges:
  (N + 64) u32 A, for numerator and denominator each.
* p_j rounded to 16 bits before the product (16-bit types): u A.
* The result's own rounding: u |o|, plus half of fp16's smallest step, and 2^-126
  for bf16 and fp32: results below the smallest normal number may be flushed.
"""
import math

import torch


def visible(pos, ctx, window, sinks):
    """bool [rows, ctx] for rows at positions pos."""
    p = torch.as_tensor(pos)[:, None]
    j = torch.arange(ctx)[None]
    ok = j <= p
    if window:
        ok = ok & ((p - j < window) | (j < sinks))
    return ok


def e8m0(x):
    return torch.exp2(x.view(torch.uint8).double() - 127)


def quantise(x):
    """(values, scale) in float64 of rows x (any float type), by the format's definition."""
    x = x.double()
    top = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for _ in range(400):  # smallest power of two with top <= 448 * 2^e
        more = top > 448 * torch.exp2(e)
        if not bool(more.any()):
            break
        e = e + more
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.round(y / step) * step
    q = torch.where(x.isfinite(), q, torch.full_like(q, math.nan))
    return q, torch.exp2(e).squeeze(-1)


def attention(q, k_cache, v_cache, block_tables, context_lens, cu, *, window=None, sinks=0, k_scale=None,
              v_scale=None, scale=None, max_seqlen_q=None):
    """(o, tolerance, lse, lse tolerance) in float64: [T, Hq, D] and [Hq, T];
    rows that are not computed hold NaN."""
    T, Hq, D = q.shape
    nb, Hkv, bs, _ = k_cache.shape
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    u32 = 2.0 ** -24
    floor = 2.0 ** (-25 if dt == torch.float16 else -126)
    o, tol = torch.full((2, T, Hq, D), math.nan, dtype=torch.float64)
    lse, ltol = torch.full((2, Hq, T), math.nan, dtype=torch.float64)
    for s, ln in enumerate(context_lens.tolist()):
        a, b = (s, s + 1) if cu is None else (int(cu[s]), int(cu[s + 1]))
        n, done = b - a, min(b - a, max_seqlen_q if max_seqlen_q is not None else b - a)
        ctx = min(max(ln, 0), block_tables.shape[1] * bs)
        ids = block_tables[s].long()[torch.arange(ctx) // bs]
        there = (ids >= 0) & (ids < nb)
        at = ids.clamp(0, nb - 1), torch.arange(ctx) % bs
        k = k_cache[at[0], :, at[1]].double()  # [ctx, Hkv, D]
        v = v_cache[at[0], :, at[1]].double()
        if k_scale is not None:
            k = k * e8m0(k_scale)[at[0], :, at[1]][..., None]
            v = v * e8m0(v_scale)[at[0], :, at[1]][..., None]
        ok = visible(max(ln, 0) - n + torch.arange(done), ctx, window, sinks) & there
        used = ok.any(0)  # cached values no row sees must not matter
        k, v = (torch.where(used[:, None, None], x, torch.zeros_like(x)) for x in (k, v))
        for h in range(Hq):
            qh, kh, vh = q[a:a + done, h].double(), k[:, h // G], v[:, h // G]
            x = (qh @ kh.T * scale).masked_fill(~ok, -math.inf)
            mx = x.amax(-1, keepdim=True) if ctx else torch.full((done, 1), -math.inf, dtype=torch.float64)
            p = torch.exp(x - mx.clamp(min=-1e300))
            total = p.sum(-1, keepdim=True)
            inv = torch.where(total > 0, 1 / total, torch.zeros_like(total))
            out, A = p @ vh * inv, p @ vh.abs() * inv
            dots = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(~ok, 0.0)
            g = (2 * (D + 4) * u32 * dots.amax(-1, keepdim=True) if ctx else 0.0) + 2.0 ** -21
            sums = (ctx + 64) * u32
            rel = 2 * g + 2 * sums + (u if dt != torch.float32 else 0.0)
            o[a:a + done, h] = out
            tol[a:a + done, h] = (1 + 4 * u) * (u * out.abs() + rel * A) + floor
            l2 = mx + torch.log(total)
            lse[h, a:a + done] = l2.squeeze(-1)
            ltol[h, a:a + done] = (g + sums + 2.0 ** -22 * l2.abs() + 2.0 ** -22).squeeze(-1)
    return o, tol, lse, ltol


def check(got, want, tol, what="output"):
    """got within tol of want wherever want is not NaN; returns nothing."""
    got = got.double().cpu()
    m = ~want.isnan()
    assert bool(got[m].isfinite().all() | want[m].isinf().any()), f"{what}: not finite"
    same = (got == want) & m  # infinities
    off = torch.where(m & ~same, (got - want).abs() - tol, torch.full_like(want, -1.0))
    worst = off.max() if off.numel() else torch.tensor(-1.0)
    assert float(worst) <= 0, f"{what}: {int((off > 0).sum())} of {int(m.sum())} off by up to {float(worst):.3g} beyond the bound"


def build(lens, new, H, G, D, bs, dtype, *, quantised=False, seed=0, extra=5, holes=(), garbage=True, pad=0):
    """A ragged batch over a shuffled cache (CPU tensors): dict of the operator's arguments.
    holes: (sequence, page) pairs taken out of the table; garbage: cells that hold no token are NaN."""
    g = torch.Generator().manual_seed(seed)
    per = max(1, max(-(-max(l, 1) // bs) for l in lens))
    nb = sum(-(-max(l, 0) // bs) for l in lens) + extra
    perm = torch.randperm(nb, generator=g)
    bt = torch.full((len(lens), per), -1, dtype=torch.int32)
    k, v = (torch.randn(nb, H, bs, D, generator=g).to(dtype) for _ in range(2))
    live = torch.zeros(nb, bs, dtype=torch.bool)
    at = 0
    for s, l in enumerate(lens):
        n = -(-max(l, 0) // bs)
        bt[s, :n] = perm[at:at + n].to(torch.int32)
        at += n
        for i in range(n):
            live[bt[s, i].long(), : min(bs, l - i * bs)] = True
    for s, i in holes:
        bt[s, i] = -1 if i % 2 else nb + 3
    ks = vs = None
    if quantised:
        (k, ks), (v, vs) = ((q.float().to(torch.float8_e4m3fn), e.to(torch.float8_e8m0fnu))
                            for q, e in (quantise(k), quantise(v)))
    if garbage:
        bad = torch.tensor(math.nan).to(k.dtype)
        for c in (k, v):
            raw, b = (c.view(torch.uint8), bad.view(torch.uint8)) if quantised else (c, bad)
            raw[(~live)[:, None, :].expand(nb, H, bs)] = b
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    q = torch.randn(int(cu[-1]) + pad, H * G, D, generator=g).to(dtype)
    return {"q": q, "k_cache": k, "v_cache": v, "block_tables": bt,
            "context_lens": torch.tensor(lens, dtype=torch.int32), "cu": cu, "most": max(new),
            "k_scale": ks, "v_scale": vs}
