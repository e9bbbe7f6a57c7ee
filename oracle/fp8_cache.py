"""64-bit restatement of the 8-bit KV cache (test infrastructure only, see oracle/__init__.py): the rounding scatter of
include/nvattn.h's nva_store_kvcache_fp8, one token and one head at a time, and attention over the values the cache
stands for, with a bound on what the kernel may be off."""
import math

import torch

E4M3_MAX = 448.0


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """float64 -> nearest e4m3 value (ties to even), clamped to 448; NaN and infinities to NaN."""
    bad = ~torch.isfinite(x)
    a = torch.where(bad, torch.zeros_like(x), x).abs().clamp(max=E4M3_MAX)
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    r = torch.round(a / step) * step          # torch.round: half to even
    r = torch.copysign(r.clamp(max=E4M3_MAX), x)
    return torch.where(bad, torch.full_like(x, math.nan), r)


def scale_of(amax: float) -> float:
    """2^e, e the least whole number with amax <= 448 * 2^e, kept in [-40, 40]."""
    if amax == 0:
        return 2.0 ** -40
    e = -40
    while e < 40 and amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def store_ref(rows, cache, scale, slots):
    """rows [T, KVH, D] into cache [NB, BS, KVH, D] (float8_e4m3fn, CPU) and scale [NB, KVH, BS / G], in place."""
    NB, BS, KVH, D = cache.shape
    blocks = scale.shape[2]
    G = BS // blocks
    flat = cache.view(NB * blocks, G, KVH, D)
    last = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < NB * BS:
            last.setdefault(s // G, {})[s % G] = i
    for b, members in last.items():
        page, j = divmod(b, blocks)
        for h in range(KVH):
            new = {s: rows[i, h].double() for s, i in members.items()}
            amax = max(float(torch.where(torch.isfinite(v), v, torch.zeros_like(v)).abs().max()) for v in new.values())
            old = float(scale[page, h, j])
            now = scale_of(amax) if 0 in members else max(old, scale_of(amax))
            if 0 not in members and now > old:
                held = flat[b, :, h].double() * (old / now)
                flat[b, :, h] = e4m3(held).to(torch.float8_e4m3fn)
            for s, v in new.items():
                flat[b, s, h] = e4m3(v / now).float().to(torch.float8_e4m3fn)
            scale[page, h, j] = now


def values(cache: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What an 8-bit cache stands for, float64 [NB, BS, KVH, D]."""
    NB, BS, KVH, D = cache.shape
    s = scale.double().transpose(1, 2).repeat_interleave(BS // scale.shape[2], dim=1)
    return cache.double() * s[..., None]


def attention_ref(q, k, v, scale):
    """q [n, H, D], k / v [L, KVH, D] (float64) -> (out, bound) [n, H, D], causal from the bottom right.

    The bound, per element: the output is rounded to bf16 (half a step, 2^-8 relative).  The kernels' weights are
    rounded to bf16 (long runs: half a step, 2^-8 of a weight, as its leading bit may be the least) or to float16, kept
    as three e5m2 parts (short runs: 2^-11), so the weighted sum is off by at most 2^-8 of sum p |v|; the parts' smallest
    step is 2^-16 where the row's largest weight is 2^12 at least: half of it, 2^-29 of the largest, for each token, times
    the largest |v|.  Scores are float32 sums of 128 products (exact where a row's values lie within 2^10 of each other):
    off by at most 130 * 2^-24 of sum |q k| (in natural units after the scale), and the exponential and the running sums
    by 2^-20."""
    n, H, D = q.shape
    L, KVH, _ = k.shape
    G = H // KVH
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if L == 0:
        return out, bound
    i = torch.arange(n, device=q.device)[:, None]
    hidden = torch.arange(L, device=q.device)[None, :] > L - n + i
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        s = q[:, h] @ kh.T * scale
        s = s.masked_fill(hidden, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        out[:, h] = p @ vh
        mass = p @ vh.abs()
        score = 130 * 2.0 ** -24 * scale * (q[:, h].abs() @ kh.abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True)
        big = vh.abs().amax() * p.amax(-1, keepdim=True)
        bound[:, h] = 2.0 ** -8 * out[:, h].abs() + (2.0 ** -8 + 2 * score + 2.0 ** -20) * mass + L * 2.0 ** -29 * big
    return out, bound + 1e-30


def paged_ref(q, cache, scales, lens, table, scale, starts=None):
    """The paged call on one device in float64: q [B, n, H, D], or [T, H, D] with starts [B + 1]."""
    flat = q.double().reshape(-1, q.shape[-2], q.shape[-1])
    out, bound = torch.zeros_like(flat), torch.zeros_like(flat)
    BS = cache[0].shape[1]
    n = q.shape[1]
    for b, L in enumerate(lens):
        r0, r1 = (starts[b], starts[b + 1]) if starts is not None else (b * n, (b + 1) * n)
        if L <= 0 or r1 == r0:
            continue
        pages = table[b, :(L + BS - 1) // BS].long()
        kv = [values(c.view(torch.uint8)[pages].view(torch.float8_e4m3fn), s[pages]).flatten(0, 1)[:L]
              for c, s in zip(cache, scales)]
        out[r0:r1], bound[r0:r1] = attention_ref(flat[r0:r1], kv[0], kv[1], scale)
    return out.view(q.shape), bound.view(q.shape)
