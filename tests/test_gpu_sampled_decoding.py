"""The four operators as a serving step uses them: Attention.forward over an 8-bit cache through prefill, decode and
verify steps, then sampling and speculative sampling on the logits; each stage against its float64 restatement on what
the stage before gave."""
import numpy as np
import pytest
import torch

from oracle import fp8_cache, sampling

pytestmark = pytest.mark.gpu

H, KVH, D, V, BS = 8, 2, 128, 997, 256


def test_speculative_steps_over_an_8_bit_cache(cuda):
    from nvattn import ops, sampler
    from nvattn.attention import Attention
    from nvattn.context import reset_context, set_context
    g = torch.Generator().manual_seed(0)
    prompts, k = [270, 40, 513], 2
    S = len(prompts)
    attn = Attention(H, D, D ** -0.5, KVH)
    NB = 12
    attn.k_cache, attn.v_cache = (torch.zeros(NB, BS, KVH, D, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    attn.k_scale, attn.v_scale = ops.kvcache_scales(attn.k_cache)
    rc = [torch.zeros(NB, BS, KVH, D, dtype=torch.float8_e4m3fn) for _ in range(2)]
    rs = [torch.zeros(NB, KVH, BS // 16) for _ in range(2)]
    table = torch.randperm(NB, generator=g)[:S * 3].view(S, 3).int()
    embed = torch.randn(V, H * D, generator=g).cuda().bfloat16()
    head = (torch.randn(V, H * D, generator=g) * 0.2).cuda().bfloat16()
    kv = (torch.randn(2, V, KVH * D, generator=g) * 0.7).cuda().bfloat16()

    def step(tokens, lens, new, prefill):
        """tokens: the step's new token ids, all sequences in a row; lens: context including them."""
        rows = [(b, p) for b in range(S) for p in range(lens[b] - new[b], lens[b])]
        slots = torch.tensor([int(table[b, p // BS]) * BS + p % BS for b, p in rows], dtype=torch.int32)
        q = embed[tokens].view(-1, H, D)
        key, value = kv[0][tokens].view(-1, KVH, D), kv[1][tokens].view(-1, KVH, D)
        cu = lambda x: torch.tensor([0] + list(x)).cumsum(0).int().cuda()  # noqa: E731
        if prefill:
            set_context(True, cu(new), cu(lens), max(new), max(lens), slots.cuda(), None, table.cuda())
        else:
            set_context(False, slot_mapping=slots.cuda(), context_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                        block_tables=table.cuda())
        o = attn(q, key, value)
        reset_context()
        for i, x in enumerate((key, value)):
            fp8_cache.store_ref(x.cpu(), rc[i], rs[i], slots)
        for c, s, r, t in zip((attn.k_cache, attn.v_cache), (attn.k_scale, attn.v_scale), rc, rs):
            assert torch.equal(c.cpu().view(torch.uint8), r.view(torch.uint8)) and torch.equal(s.cpu(), t)
        want, bound = fp8_cache.paged_ref(q.cpu(), rc, rs, lens, table, attn.scale, cu(new).tolist())
        assert ((o.cpu().double() - want).abs() <= bound).all()
        return o.view(len(rows), H * D)

    lens = list(prompts)
    text = [torch.randint(0, V, (n,), generator=g).tolist() for n in prompts]
    # the prompt in two prefill chunks (the second over the cached first)
    half = [n // 2 for n in prompts]
    step(torch.tensor(sum((t[:h] for t, h in zip(text, half)), [])).cuda(), half, half, True)
    rest = [n - h for n, h in zip(prompts, half)]
    o = step(torch.tensor(sum((t[h:] for t, h in zip(text, half)), [])).cuda(), lens, rest, True)
    last = torch.tensor(rest).cumsum(0) - 1
    t = torch.tensor([0.0, 0.8, 1.1])
    settings = dict(top_k=torch.tensor([0, 50, 0], dtype=torch.int32), top_p=torch.tensor([1.0, 0.95, 0.9]),
                    min_p=torch.tensor([0.0, 0.0, 0.02]))
    dev = {n: x.cuda() for n, x in settings.items()}
    logits = o[last.cuda()] @ head.T
    u = torch.rand(S, generator=g)
    ids = sampler.sample_tokens(logits, t.cuda(), u.cuda(), **dev).cpu()
    host = logits.float().cpu().numpy()
    for s in range(S):
        assert int(ids[s]) == sampling.sample(host[s], float(t[s]), float(u[s]),
                                              *(settings[n][s].item() for n in ("top_k", "top_p", "min_p")))[0]
    total = 0
    for it in range(6):
        # each sequence brings its last token and k drafts; rejected drafts' slots are written again by the next step
        drafts = torch.randint(0, V, (S, k), generator=g)
        if it % 2:                                   # likely drafts: the greedy tokens of the logits before
            drafts[:, 0] = torch.from_numpy(host.reshape(S, -1, V)[:, -1].argmax(-1))
        num = torch.tensor([k, k, 1])
        tokens = torch.cat([ids[:, None], drafts], 1)
        lens = [n + k + 1 for n in lens]
        o = step(tokens.reshape(-1).cuda(), lens, [k + 1] * S, False)
        logits = o @ head.T
        au, u = torch.rand(S, k, generator=g) * 0.2, torch.rand(S, generator=g)
        a, nxt = sampler.verify_drafts_sampled(logits, drafts.cuda(), num.cuda(), t.cuda(), au.cuda(), u.cuda(), **dev)
        host = logits.float().cpu().numpy()
        for s in range(S):
            want = sampling.verify(host.reshape(S, k + 1, V)[s], drafts[s].tolist(), int(num[s]), float(t[s]),
                                   au[s].double().tolist(), float(u[s]),
                                   *(settings[n][s].item() for n in ("top_k", "top_p", "min_p")))
            assert (int(a[s]), int(nxt[s])) == want
        ids = nxt.cpu()
        lens = [n - k + int(a[s]) for s, n in enumerate(lens)]
        total += int(a.sum())
    assert np.isfinite(host).all()


def test_prefill_without_a_block_table_attends_over_its_own_rows(cuda):
    """The first prefill of a batch (no prefix): bf16 attention over the step's K/V, 8-bit rows stored on the side."""
    from nvattn import ops
    from nvattn.attention import Attention
    from nvattn.context import reset_context, set_context
    g = torch.Generator().manual_seed(1)
    q, key, value = (torch.randn(130, n, D, generator=g).bfloat16() for n in (H, KVH, KVH))
    outs = []
    for fp8 in (False, True):
        attn = Attention(H, D, D ** -0.5, KVH)
        dt = torch.float8_e4m3fn if fp8 else torch.bfloat16
        attn.k_cache, attn.v_cache = (torch.zeros(2, BS, KVH, D, dtype=dt, device="cuda") for _ in range(2))
        if fp8:
            attn.k_scale, attn.v_scale = ops.kvcache_scales(attn.k_cache, 64)
        cu = torch.tensor([0, 130], dtype=torch.int32, device="cuda")
        set_context(True, cu, cu, 130, 130, torch.arange(130, dtype=torch.int32, device="cuda"))
        outs.append(attn(q.cuda(), key.cuda(), value.cuda()))
        reset_context()
    assert torch.equal(outs[0], outs[1])
    rc, rs = torch.zeros(2, BS, KVH, D, dtype=torch.float8_e4m3fn), torch.zeros(2, KVH, 4)
    fp8_cache.store_ref(key, rc, rs, torch.arange(130))
    assert torch.equal(attn.k_cache.cpu().view(torch.uint8), rc.view(torch.uint8)) and torch.equal(attn.k_scale.cpu(), rs)
