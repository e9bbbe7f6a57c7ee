"""The fused prologue's choice between its own KV scatter and the 8-bit cache's (nvattn.nanovllm_dropin,
install_fused_prologue), without a GPU: nano-vllm's modules and the two ops are stand-ins that record their calls."""
import sys
import types

import pytest
import torch

H, KVH, D, T = 4, 2, 128, 5


@pytest.fixture()
def attention(monkeypatch):
    """A Qwen3Attention stand-in with the prologue installed: (layer, context, calls)."""
    from nvattn import nanovllm_dropin, ops
    context = types.SimpleNamespace(is_prefill=False, block_tables=torch.zeros(1, 1), slot_mapping=torch.arange(T))
    calls = []

    class Qwen3Attention:
        pass

    qwen3 = types.ModuleType("nanovllm.models.qwen3")
    qwen3.Qwen3Attention = Qwen3Attention
    names = {"nanovllm": types.ModuleType("nanovllm"), "nanovllm.models": types.ModuleType("nanovllm.models"),
             "nanovllm.models.qwen3": qwen3, "nanovllm.utils": types.ModuleType("nanovllm.utils"),
             "nanovllm.utils.context": types.ModuleType("nanovllm.utils.context")}
    names["nanovllm.utils.context"].get_context = lambda: context
    names["nanovllm.models"].qwen3 = qwen3
    for name, module in names.items():
        monkeypatch.setitem(sys.modules, name, module)
    monkeypatch.setattr(nanovllm_dropin, "_installed", {"attention"})

    def prologue(qkv, positions, cos_sin, qw, kw, eps, heads, kv_heads, k_cache, v_cache, slots, want_k=False):
        calls.append(("prologue", k_cache, v_cache, slots, want_k))
        return "q", "k" if want_k else None, "v"

    monkeypatch.setattr(ops, "qk_norm_rope_store", prologue)
    monkeypatch.setattr(ops, "store_kvcache", lambda *a: calls.append(("store",) + a))
    nanovllm_dropin.install_fused_prologue()
    layer = Qwen3Attention()
    layer.qkv_bias, layer.num_heads, layer.num_kv_heads = False, H, KVH
    layer.qkv_proj, layer.post_attn = (lambda x: x), (lambda o: o)
    layer.rotary_emb = types.SimpleNamespace(cos_sin_cache=None)
    layer.q_norm = layer.k_norm = types.SimpleNamespace(weight=None, eps=1e-6)

    def forward_stored(q, k, v):
        calls.append(("attend", q, k, v))
        return "o"

    layer.attn = types.SimpleNamespace(k_cache=torch.zeros(2, 256, KVH, D), v_cache=torch.ones(2, 256, KVH, D),
                                       k_scale=None, v_scale=None, forward_stored=forward_stored)
    return layer, context, calls


@pytest.mark.parametrize("is_prefill,paged", [(False, True), (True, True), (True, False)])
def test_8_bit_cache_is_written_by_its_own_scatter(attention, is_prefill, paged):
    """The prologue gets no cache and gives k; the rounding scatter gets both with the scales; then the attention."""
    layer, context, calls = attention
    context.is_prefill, context.block_tables = is_prefill, torch.zeros(1, 1) if paged else None
    a = layer.attn
    a.k_scale, a.v_scale = torch.zeros(1), torch.ones(1)
    assert layer.forward(None, torch.zeros(T, 8)) == "o"
    prologue, store, attend = calls
    assert prologue == ("prologue", None, None, None, True)
    assert store[0] == "store" and store[1:3] == ("k", "v") and store[3] is a.k_cache and store[4] is a.v_cache
    assert store[5] is context.slot_mapping and store[6] is a.k_scale and store[7] is a.v_scale
    assert attend == ("attend", "q", "k", "v")


@pytest.mark.parametrize("is_prefill,paged", [(False, True), (True, True), (True, False)])
def test_bf16_cache_is_written_by_the_prologue(attention, is_prefill, paged):
    layer, context, calls = attention
    context.is_prefill, context.block_tables = is_prefill, torch.zeros(1, 1) if paged else None
    layer.forward(None, torch.zeros(T, 8))
    prologue, attend = calls
    assert prologue[1] is layer.attn.k_cache and prologue[2] is layer.attn.v_cache
    assert prologue[3] is context.slot_mapping and prologue[4] == (is_prefill and not paged)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_without_a_cache_or_a_scatter_nothing_is_stored(attention, eight_bit):
    """Warm-up (the caches are not there yet) and the pieces of a mixed step (the attention module stores)."""
    layer, context, calls = attention
    if eight_bit:
        layer.attn.k_scale = layer.attn.v_scale = torch.ones(1)
    assert layer.pre_attn(None, torch.zeros(T, 8)) == ("q", "k", "v")
    layer.attn.k_cache = layer.attn.v_cache = torch.tensor([])
    context.is_prefill, context.block_tables = True, None
    layer.forward(None, torch.zeros(T, 8))
    assert [c[0] for c in calls] == ["prologue", "prologue", "attend"]
    assert all(c[1] is None and c[4] for c in calls[:2])
