"""What a sampled decode step over an 8-bit KV cache computes, as measurable cases.

Four operators, in the order a serving step meets them:

  store    this step's K/V rows into a paged cache of e4m3 values with one float32 scale (a power of two) for each
           block of consecutive tokens and kv head
  attend   decode / verify / mixed varlen attention over that cache
  sample   one token per row of logits, with temperature, top-k, top-p and min-p, from given uniform numbers
  verify   speculative sampling: how many fixed drafts of each sequence are accepted, and the token after them

`own` chooses between the plain forms written out here (elementary torch operations) and the calls a user makes.
"""
import math
import os
import sys

import torch

own = False

HEAD_DIM = 128
PAGE = 256
E4M3_MAX = 448.0
EXP_MIN, EXP_MAX = -40, 40


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 sequences: every row lands in a partly filled block of its own
        {"name": "store decode 64", "op": "store", "tokens": 64, "runs": 64, "kv_heads": 8, "scale_block": 16},
        # a prefill of eight 1024-token prompts: whole blocks, bandwidth
        {"name": "store prefill 8192", "op": "store", "tokens": 8192, "runs": 8, "kv_heads": 8, "scale_block": 16},
        # the smallest decode: four short sequences of a 16 / 8-head model, latency
        {"name": "attend decode 4 short", "op": "attend", "mode": "decode", "seqs": 4, "lo": 37, "hi": 1000, "n": 1,
         "heads": 16, "kv_heads": 8, "scale_block": 16},
        # an ordinary decode batch: 64 sequences, contexts 512 to 4096
        {"name": "attend decode 64", "op": "attend", "mode": "decode", "seqs": 64, "lo": 512, "hi": 4096, "n": 1,
         "heads": 32, "kv_heads": 8, "scale_block": 16},
        # the verify step of speculative decoding: four drafts, contexts 256 to 2048, coarser scales
        {"name": "attend verify k4", "op": "attend", "mode": "decode", "seqs": 32, "lo": 256, "hi": 2048, "n": 5,
         "heads": 32, "kv_heads": 8, "scale_block": 128},
        # a mixed step under a 2048-token budget: three prefill chunks over cached prefixes next to 256 decode rows
        {"name": "attend mixed", "op": "attend", "mode": "varlen", "seqs": 256, "lo": 16, "hi": 4096, "n": 1,
         "chunks": 3, "chunk": 597, "prefix": 427, "heads": 32, "kv_heads": 8, "scale_block": 16},
        # long contexts: eight sequences of up to 65,536 tokens
        {"name": "attend decode long", "op": "attend", "mode": "decode", "seqs": 8, "lo": 40000, "hi": 65536, "n": 1,
         "heads": 32, "kv_heads": 8, "scale_block": 64},
        # one sequence's next token: latency
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "bfloat16", "params": "mixed"},
        # an ordinary batch where each request has its own settings (temperature 0 among them)
        {"name": "sample 64 mixed", "op": "sample", "rows": 64, "vocab": 151936, "dtype": "float32",
         "params": "mixed"},
        # the largest batch, temperature alone: every token of the vocabulary stays in
        {"name": "sample 510 plain", "op": "sample", "rows": 510, "vocab": 151936, "dtype": "bfloat16",
         "params": "temperature"},
        # speculative sampling of four sequences with two drafts
        {"name": "verify 4 k2", "op": "verify", "seqs": 4, "k": 2, "vocab": 151936, "dtype": "bfloat16",
         "params": "mixed"},
        # speculative sampling of 32 sequences with four drafts
        {"name": "verify 32 k4", "op": "verify", "seqs": 32, "k": 4, "vocab": 151936, "dtype": "bfloat16",
         "params": "mixed"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "sample", "verify"])
    if op == "store":
        tokens = _log_int(rng, 1, 8192)
        return {"op": op, "tokens": tokens, "runs": _log_int(rng, 1, min(tokens, 256)),
                "kv_heads": rng.choice([1, 2, 4, 8]), "scale_block": rng.choice([8, 16, 32, 64, 128, 256])}
    if op == "attend":
        heads, kv_heads = rng.choice([(32, 8), (16, 8), (16, 4), (8, 2), (8, 1), (4, 4), (40, 8)])
        scale_block = rng.choice([16, 32, 64, 128, 256])
        seqs = _log_int(rng, 1, 200)
        hi = _log_int(rng, 64, min(65536, 262144 // seqs))
        lo = _log_int(rng, 1, hi)
        if rng.random() < 0.3:
            chunk = _log_int(rng, 2, 600)
            return {"op": op, "mode": "varlen", "seqs": min(seqs, 64), "lo": min(lo, 1024), "hi": min(hi, 4096), "n": 1,
                    "chunks": rng.randint(1, 3), "chunk": chunk, "prefix": _log_int(rng, 1, 1000), "heads": heads,
                    "kv_heads": kv_heads, "scale_block": scale_block}
        return {"op": op, "mode": "decode", "seqs": seqs, "lo": lo, "hi": hi,
                "n": rng.choice([1, 1, 1, 2, 3, 5, 9]) if heads // kv_heads <= 5 else rng.choice([1, 3, 6]),
                "heads": heads, "kv_heads": kv_heads, "scale_block": scale_block}
    vocab = rng.choice([151936, _log_int(rng, 100, 151936), _log_int(rng, 1000, 151936)])
    case = {"op": op, "vocab": vocab, "dtype": rng.choice(["bfloat16", "float32"]),
            "params": rng.choice(["mixed", "mixed", "temperature", "top_k", "top_p", "min_p"])}
    if op == "sample":
        return {**case, "rows": _log_int(rng, 1, 250)}
    k = rng.choice([1, 2, 3, 4, 8])
    return {**case, "k": k, "seqs": _log_int(rng, 1, max(1, 250 // (k + 1)))}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rand(g, *shape, dtype=torch.float32):
    return torch.rand(*shape, generator=g, device="cuda", dtype=dtype)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _host_ints(seed, n, lo, hi):
    g = torch.Generator().manual_seed(int(seed) * 7919 + 1)
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def _scales(e):
    """2^e as float32, for whole e."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e.to(torch.int32))


def _exponent(amax):
    """The least whole e with amax <= 448 * 2^e, kept in [-40, 40]."""
    f, k = torch.frexp(amax.float())
    e = torch.where(2 * f <= E4M3_MAX / 256, k - 9, k - 8)
    return torch.where(amax > 0, e, torch.full_like(e, EXP_MIN)).clamp(EXP_MIN, EXP_MAX)


def _filled_cache(g, pages, kv_heads, block, size):
    """A cache whose pages hold earlier tokens: values around `size`, one scale per (page, head, block of tokens)."""
    x = (_randn(g, pages, PAGE // block, block, kv_heads, HEAD_DIM) * size).to(torch.bfloat16).float()
    e = _exponent(x.abs().amax(dim=(2, 4)))                                   # [pages, blocks, heads]
    x.mul_(_scales(-e)[:, :, None, :, None])
    c = x.to(torch.float8_e4m3fn).view(pages, PAGE, kv_heads, HEAD_DIM)
    return c, _scales(e).transpose(1, 2).contiguous()                         # scales [pages, heads, blocks]


def _prepare_store(case, seed):
    g = _gen(seed)
    T, runs, kvh, block = case["tokens"], case["runs"], case["kv_heads"], case["scale_block"]
    # `runs` sequences append T tokens between them: each writes consecutive positions into pages of its own
    share = [T // runs + (1 if i < T % runs else 0) for i in range(runs)]
    first = _host_ints(seed, runs, 0, PAGE - 1) if T < 4 * runs else [0] * runs
    need = [(f + n + PAGE - 1) // PAGE for f, n in zip(first, share)]
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    slots, at = [], 0
    for f, n, w in zip(first, share, need):
        mine = order[at:at + w]
        at += w
        slots += [mine[(f + i) // PAGE] * PAGE + (f + i) % PAGE for i in range(n)]
    k_cache, k_scale = _filled_cache(g, pages, kvh, block, 0.5)
    v_cache, v_scale = _filled_cache(g, pages, kvh, block, 0.5)
    # the rows come as column slices of the fused projection's output, some tokens louder than what the blocks hold
    qkv = _randn(g, T, 4 * kvh * HEAD_DIM) * (0.25 + _rand(g, T, 1))
    qkv = qkv.to(torch.bfloat16)
    return {"key": qkv[:, 2 * kvh * HEAD_DIM:3 * kvh * HEAD_DIM].view(T, kvh, HEAD_DIM),
            "value": qkv[:, 3 * kvh * HEAD_DIM:].view(T, kvh, HEAD_DIM), "k_cache": k_cache, "v_cache": v_cache,
            "k_scale": k_scale, "v_scale": v_scale, "slots": torch.tensor(slots, dtype=torch.int32, device="cuda")}


def _prepare_attend(case, seed):
    g = _gen(seed)
    H, kvh, block, n = case["heads"], case["kv_heads"], case["scale_block"], case["n"]
    lens = _host_ints(seed, case["seqs"], case["lo"], case["hi"])
    qlens = [n] * case["seqs"]
    if case["mode"] == "varlen":
        qlens = [case["chunk"] + 7 * i for i in range(case["chunks"])] + qlens
        lens = [q + case["prefix"] * i for i, q in enumerate(qlens[:case["chunks"]])] + lens
    else:
        lens = [max(x, n) if case["seqs"] < 3 or i % 61 != 60 else 0 for i, x in enumerate(lens)]
    pages_of = [(x + PAGE - 1) // PAGE for x in lens]
    pages = sum(pages_of) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    width = max(1, max(pages_of))
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for i, w in enumerate(pages_of):
        table[i, :w] = torch.tensor(order[at:at + w], dtype=torch.int32)
        at += w
    k_cache, k_scale = _filled_cache(g, pages, kvh, block, 1.0)
    v_cache, v_scale = _filled_cache(g, pages, kvh, block, 0.5)
    q = _randn(g, sum(qlens), H, HEAD_DIM).to(torch.bfloat16)
    cu = lambda xs: torch.tensor([0] + xs, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()  # noqa: E731
    return {"q": q if case["mode"] == "varlen" else q.view(len(lens), n, H, HEAD_DIM), "k_cache": k_cache,
            "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale, "table": table.cuda(),
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cu_q": cu(qlens), "cu_k": cu(lens),
            "max_q": max(qlens), "max_k": max(lens), "scale": HEAD_DIM ** -0.5, "n": n,
            "chunks": case.get("chunks", 0) if case["mode"] == "varlen" else 0}


def _settings(case, seed, rows):
    g = _gen(seed + 17)
    kind = case["params"]
    pick = lambda xs: torch.tensor(xs, device="cuda")[torch.randint(len(xs), (rows,), generator=g, device="cuda")]  # noqa: E731
    t = pick([0.6, 0.7, 0.8, 1.0, 1.0, 1.3])
    if kind == "mixed" and rows > 1:
        t = torch.where(torch.arange(rows, device="cuda") % 8 == 3, torch.zeros_like(t), t)
    on = lambda name: kind == "mixed" or kind == name  # noqa: E731
    return {"temperatures": t.float(),
            "top_k": pick([0, 20, 50, 1000]).to(torch.int32) if on("top_k") else None,
            "top_p": pick([0.8, 0.9, 0.95, 1.0]).float() if on("top_p") else None,
            "min_p": pick([0.0, 0.0, 0.02, 0.1]).float() if on("min_p") else None}


def _logits(case, seed, rows):
    g = _gen(seed)
    x = _randn(g, rows, case["vocab"]) * 2.5
    # a few likely tokens stand out of the bulk, as a language model's do
    top = torch.randint(case["vocab"], (rows, 12), generator=g, device="cuda")
    x.scatter_add_(1, top, 6.0 + 4.0 * _randn(g, rows, 12))
    return x.to(getattr(torch, case["dtype"])), g


def _prepare_sample(case, seed):
    x, g = _logits(case, seed, case["rows"])
    return {"logits": x, "uniforms": _rand(g, case["rows"]), **_settings(case, seed, case["rows"])}


def _prepare_verify(case, seed):
    S, K = case["seqs"], case["k"]
    x, g = _logits(case, seed, S * (K + 1))
    # drafts that are often the likely token, as a good proposer's are
    likely = x.view(S, K + 1, -1)[:, :K].float().argmax(-1)
    other = torch.randint(case["vocab"], (S, K), generator=g, device="cuda")
    drafts = torch.where(_rand(g, S, K) < 0.8, likely, other)
    num = torch.where(_rand(g, S) < 0.7, torch.full((S,), K, device="cuda"),
                      torch.randint(0, K + 1, (S,), generator=g, device="cuda"))
    return {"logits": x, "drafts": drafts, "num_drafts": num, "accept_uniforms": _rand(g, S, K),
            "uniforms": _rand(g, S), **_settings(case, seed, S)}


def prepare(case, seed):
    state = {"store": _prepare_store, "attend": _prepare_attend, "sample": _prepare_sample,
             "verify": _prepare_verify}[case["op"]](case, seed)
    return {"op": case["op"], "mode": case.get("mode"), **state}


# ------------------------------------------------------------------------------------------------ plain forms
def _store_one(x, cache, scale, slots):
    """x [T, heads, 128] into cache [pages, 256, heads, 128] (e4m3) with scale [pages, heads, blocks].  A block's
    scale is that of its largest value, a power of two; it grows with the values written, and what the block held is
    rounded again to the larger scale; a write to a block's first slot starts the block afresh."""
    pages, heads, blocks = scale.shape
    block = PAGE // blocks
    live = slots >= 0
    slots, x = slots[live].long(), x[live].float()
    at = slots // PAGE * blocks + slots % PAGE // block                        # scale block of each token
    amax = torch.zeros(pages * blocks, heads, device=x.device)
    amax.scatter_reduce_(0, at[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    touched = torch.zeros(pages * blocks, dtype=torch.bool, device=x.device)
    touched[at] = True
    fresh = torch.zeros_like(touched)
    fresh[at[slots % block == 0]] = True
    old = scale.transpose(1, 2).reshape(pages * blocks, heads)
    e = _scales(_exponent(amax))
    new = torch.where(touched[:, None], torch.where(fresh[:, None], e, torch.maximum(e, old)), old)
    grown = touched & ~fresh
    ids = grown.nonzero()[:, 0]
    held = cache.view(torch.uint8).view(pages * blocks, block, heads, HEAD_DIM)
    was = held[ids].view(torch.float8_e4m3fn).float() * (old[ids] / new[ids])[:, None, :, None]
    held[ids] = was.to(torch.float8_e4m3fn).view(torch.uint8)
    y = (x / new[at][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    cache.view(torch.uint8).view(-1, heads, HEAD_DIM)[slots] = y.to(torch.float8_e4m3fn).view(torch.uint8)
    scale.copy_(new.view(pages, blocks, heads).transpose(1, 2))


def _gathered(cache, scale, table, width, wide=torch.float32):
    """The pages of `table` [B, W] as [B, width, heads, 128], scaled."""
    pages, heads, blocks = scale.shape
    ids = table.clamp(min=0).long()[:, :(width + PAGE - 1) // PAGE]
    x = cache.view(torch.uint8)[ids].view(torch.float8_e4m3fn).to(wide)
    s = scale[ids].to(wide).transpose(2, 3).repeat_interleave(PAGE // blocks, dim=2)
    return (x * s[..., None]).flatten(1, 2)[:, :width]


def _attend_group(q, lens, table, state, width):
    """q [B, n, H, 128] over the first lens[b] cached tokens, causal from the bottom right."""
    B, n, H, D = q.shape
    heads = state["k_cache"].shape[2]
    k = _gathered(state["k_cache"], state["k_scale"], table, width)
    s = torch.matmul(q.float().view(B, n, heads, H // heads, D).permute(0, 2, 3, 1, 4).flatten(2, 3) * state["scale"],
                     k.permute(0, 2, 3, 1)).view(B, heads, H // heads, n, width)
    del k
    last = lens.view(B, 1) - n + torch.arange(n, device=q.device)              # the last visible position of each row
    seen = torch.arange(width, device=q.device) <= last[:, :, None]            # [B, n, width]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    v = _gathered(state["v_cache"], state["v_scale"], table, width).permute(0, 2, 1, 3)
    v = v * (torch.arange(width, device=q.device) < lens.view(B, 1))[:, None, :, None]
    o = torch.matmul(p.flatten(2, 3), v).view(B, heads, H // heads, n, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D).to(q.dtype)


def _attend(state):
    if state["mode"] != "varlen":
        return _attend_group(state["q"], state["lens"].long(), state["table"], state, max(1, state["max_k"]))
    # long and short query runs apart, so that neither is padded to the other
    c, q, cu, lens = state["chunks"], state["q"], state["cu_q"].long(), state["lens"].long()
    short = state["table"].shape[0] - c
    tail = q[q.shape[0] - short:].view(short, 1, *q.shape[1:])
    o_short = _attend_group(tail, lens[c:], state["table"][c:], state, state["max_k"])
    rows = cu[1:c + 1, None] - state["max_q"] + torch.arange(state["max_q"], device=q.device)   # right-aligned runs
    real = rows >= cu[:c, None]
    o_long = _attend_group(q[rows.clamp(min=0)], lens[:c], state["table"][:c], state, state["max_k"])
    return torch.cat([o_long[real], o_short[:, 0]])


def _kept_weights(x, t, top_k, top_p, min_p):
    """The weight of every token after temperature, min-p, top-k and top-p, in 64 bits; x [R, V], settings [R]."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    t = torch.where(t > 0, t, torch.ones_like(t)).double()[:, None]
    w = torch.exp(torch.where(x == m, torch.zeros_like(x), (x - m) / t))
    if min_p is not None:
        w = torch.where(w >= min_p.double()[:, None], w, torch.zeros_like(w))
    if top_k is None and top_p is None:
        return w
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    s = w.gather(1, order)
    if top_k is not None:
        k = torch.where(top_k > 0, top_k, torch.full_like(top_k, x.shape[1]))[:, None]
        s = torch.where(torch.arange(x.shape[1], device=x.device) < k, s, torch.zeros_like(s))
    if top_p is not None:
        c = s.cumsum(-1)
        keep = (c - s) < top_p.double()[:, None] * c[:, -1:]
        keep[:, 0] = True
        s = torch.where(keep | (top_p >= 1)[:, None], s, torch.zeros_like(s))
    return torch.zeros_like(w).scatter_(1, order, s)


def _drawn(w, u):
    """The first token, by index, at which the running sum of the weights passes u times their sum."""
    c = w.cumsum(-1)
    return torch.searchsorted(c, u.double()[:, None] * c[:, -1:], right=True)[:, 0]


def _sample(state):
    x, t = state["logits"], state["temperatures"]
    w = _kept_weights(x, t, state["top_k"], state["top_p"], state["min_p"])
    return torch.where(t > 0, _drawn(w, state["uniforms"]), x.float().argmax(-1))


def _verify(state):
    x, drafts, num, t = state["logits"], state["drafts"], state["num_drafts"], state["temperatures"]
    S, K = drafts.shape
    each = lambda a: None if a is None else a.repeat_interleave(K + 1)  # noqa: E731
    w = _kept_weights(x, each(t), each(state["top_k"]), each(state["top_p"]), each(state["min_p"])).view(S, K + 1, -1)
    best = x.float().argmax(-1).view(S, K + 1)
    picked = w[:, :K].gather(2, drafts[:, :, None])[:, :, 0]
    lucky = state["accept_uniforms"].double() * w[:, :K].sum(-1) < picked
    ok = torch.where(t[:, None] > 0, lucky, drafts == best[:, :K])
    ok &= torch.arange(K, device=x.device) < num[:, None]
    a = ok.long().cumprod(-1).sum(-1)
    row = torch.arange(S, device=x.device)
    last = w[row, a]
    turned = a < num                                       # the draft there was turned down: it is not drawn again
    d = drafts[row, a.clamp(max=K - 1)]
    last[row, d] = torch.where(turned, torch.zeros_like(last[row, d]), last[row, d])
    return a, torch.where(t > 0, _drawn(last, state["uniforms"]), best[row, a])


def _run_plain(state):
    op = state["op"]
    if op == "store":
        for name in ("k", "v"):
            _store_one(state["key" if name == "k" else "value"], state[name + "_cache"], state[name + "_scale"],
                       state["slots"])
        return {n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if op == "attend":
        return {"out": _attend(state)}
    if op == "sample":
        return {"ids": _sample(state)}
    a, nxt = _verify(state)
    return {"accepted": a, "next": nxt}


# ------------------------------------------------------------------------------------------------ the calls
_package = None


def _nvattn():
    global _package
    if _package is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "nano-vllm-spec-decode_b200"))
        from nvattn import ops, sampler
        _package = (ops, sampler)
    return _package


def _run_own(state):
    ops, sampler = _nvattn()
    op = state["op"]
    if op == "store":
        ops.store_kvcache(state["key"], state["value"], state["k_cache"], state["v_cache"], state["slots"],
                          k_scale=state["k_scale"], v_scale=state["v_scale"])
        return {n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if op == "attend":
        if state["mode"] == "varlen":
            return {"out": ops.flash_attn_varlen_func(
                state["q"], state["k_cache"], state["v_cache"], max_seqlen_q=state["max_q"], cu_seqlens_q=state["cu_q"],
                max_seqlen_k=state["max_k"], cu_seqlens_k=state["cu_k"], softmax_scale=state["scale"], causal=True,
                block_table=state["table"], k_scale=state["k_scale"], v_scale=state["v_scale"])}
        return {"out": ops.flash_attn_with_kvcache(
            state["q"], state["k_cache"], state["v_cache"], cache_seqlens=state["lens"], block_table=state["table"],
            softmax_scale=state["scale"], causal=True, k_scale=state["k_scale"], v_scale=state["v_scale"])}
    settings = {n: state[n] for n in ("top_k", "top_p", "min_p")}
    if op == "sample":
        return {"ids": sampler.sample_tokens(state["logits"], state["temperatures"], state["uniforms"], **settings)}
    a, nxt = sampler.verify_drafts_sampled(state["logits"], state["drafts"], state["num_drafts"],
                                           state["temperatures"], state["accept_uniforms"], state["uniforms"],
                                           **settings)
    return {"accepted": a, "next": nxt}


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case["op"] == "store":
        values = 2 * case["tokens"] * case["kv_heads"] * HEAD_DIM
        return {"bytes": 3 * values + 8 * 2 * case["kv_heads"] * max(case["runs"], case["tokens"] // case["scale_block"]),
                "flops": 2 * values}
    if case["op"] == "attend":
        n, extra_bytes, extra_flops = case["n"], 0, 0
        mean = (case["lo"] + case["hi"]) / 2
        rows, H, kvh = case["seqs"] * n, case["heads"], case["kv_heads"]
        if case["mode"] == "varlen":
            for i in range(case["chunks"]):
                qn = case["chunk"] + 7 * i
                L = qn + case["prefix"] * i
                extra_bytes += 2 * L * kvh * HEAD_DIM + 4 * qn * H * HEAD_DIM
                extra_flops += 4 * H * HEAD_DIM * qn * (L - qn / 2)
        cached = 2 * case["seqs"] * mean * kvh * HEAD_DIM * (1 + 4 / (case["scale_block"] * HEAD_DIM))
        return {"bytes": cached + 4 * rows * H * HEAD_DIM + extra_bytes,
                "flops": 4 * rows * mean * H * HEAD_DIM + extra_flops}
    rows = case["rows"] if case["op"] == "sample" else case["seqs"] * (case["k"] + 1)
    values = rows * case["vocab"]
    return {"bytes": values * (2 if case["dtype"] == "bfloat16" else 4) + 32 * rows, "flops": 4 * values}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_store(state):
    """Every written value over its block's scale, unrounded; what a block held, over its new scale."""
    slots = state["slots"].cpu().tolist()
    got = {}
    for name, rows in (("k", state["key"]), ("v", state["value"])):
        cache, scale = state[name + "_cache"], state[name + "_scale"].double()
        pages, heads, blocks = scale.shape
        block = PAGE // blocks
        value = cache.view(torch.uint8).view(torch.float8_e4m3fn).double().view(-1, heads, HEAD_DIM)
        x = rows.double()
        by_block = {}
        for i, s in enumerate(slots):
            if s >= 0:
                by_block.setdefault(s // block, []).append((s, i))
        for b, members in by_block.items():
            page, j = divmod(b, blocks)
            at = torch.tensor([i for _, i in members], device=x.device)
            biggest = x[at].abs().amax(dim=(0, 2))
            e = torch.ceil(torch.log2(biggest / E4M3_MAX)).clamp(EXP_MIN, EXP_MAX)
            new = torch.exp2(e)
            if all(s % block for s, _ in members):
                old = scale[page, :, j]
                new = torch.maximum(new, old)
                value[b * block:(b + 1) * block] *= (old / new)[None, :, None]
            scale[page, :, j] = new
            value[torch.tensor([s for s, _ in members], device=x.device)] = x[at] / new[None, :, None]
        got[name + "_cache"] = value.view(cache.shape)
        got[name + "_scale"] = scale
    return got


def _exact_attend(state):
    kvh = state["k_cache"].shape[2]
    q = state["q"].double()
    H = q.shape[-2]
    flat = q.view(-1, H, HEAD_DIM)
    lens = state["lens"].cpu().tolist()
    starts = state["cu_q"].cpu().tolist()
    out = torch.zeros_like(flat)
    for b, L in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        if not L:
            continue
        pages = state["table"][b, :(L + PAGE - 1) // PAGE].long()
        for h in range(kvh):
            kv = []
            for name in ("k", "v"):
                s = state[name + "_scale"][pages, h].double()
                c = state[name + "_cache"].view(torch.uint8)[pages, :, h].view(torch.float8_e4m3fn).double()
                kv.append((c.view(len(pages), s.shape[1], -1, HEAD_DIM) * s[:, :, None, None]).view(-1, HEAD_DIM)[:L])
            g = H // kvh
            rows = flat[r0:r1, h * g:(h + 1) * g]
            a = torch.einsum("igd,ld->igl", rows, kv[0]) * state["scale"]
            i = torch.arange(r1 - r0, device=q.device)
            hidden = torch.arange(L, device=q.device)[None, :] > (L - (r1 - r0) + i)[:, None]
            a = torch.softmax(a.masked_fill(hidden[:, None, :], float("-inf")), dim=-1)
            out[r0:r1, h * g:(h + 1) * g] = torch.einsum("igl,ld->igd", a, kv[1])
    return {"out": out.view(q.shape)}


def exact(case, seed):
    if case["op"] in ("sample", "verify"):
        return None                                  # token ids: whole numbers, held to the plain form's
    state = prepare(case, seed)
    return _exact_store(state) if case["op"] == "store" else _exact_attend(state)
