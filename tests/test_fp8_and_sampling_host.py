"""Host side of the 8-bit cache and of sampling without a GPU: what the wrappers refuse, the arguments they hand to the C
ABI, the entry points' own refusals, and the float64 restatements against torch's e4m3 and against enumeration."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import fp8_cache, sampling


class _Recorder:
    def __init__(self):
        self.calls = []

    @staticmethod
    def nva_paged_attention_fp8_workspace_bytes(n, H, KVH, D):
        return 0 if D != 128 or H // KVH > 40 else 1 << 16

    @staticmethod
    def nva_sample_workspace_bytes(rows, vocab, elem_bytes):
        return 32 * rows

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture()
def rec(monkeypatch):
    from nvattn import _lib, ops
    r = _Recorder()
    monkeypatch.setattr(_lib, "load", lambda: r)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_workspace", lambda nbytes, device: torch.zeros(max(nbytes, 16), dtype=torch.uint8))
    return r


def cache(NB=4, BS=256, KVH=8, G=16):
    from nvattn import ops
    c = torch.zeros(NB, BS, KVH, 128, dtype=torch.float8_e4m3fn)
    return c, ops.kvcache_scales(c, G)


# ---------------------------------------------------------------------------------------------- wrappers
def test_scales_layout():
    c, (ks, vs) = cache(G=64)
    assert ks.shape == vs.shape == (4, 8, 4) and ks.dtype == torch.float32 and ks.data_ptr() != vs.data_ptr()
    from nvattn import ops
    with pytest.raises(AssertionError):
        ops.kvcache_scales(c, 12)


def test_store_passes_strides_and_scale_block(rec):
    from nvattn import ops
    c, (ks, vs) = cache(G=32)
    qkv = torch.zeros(5, 48 * 128, dtype=torch.bfloat16)
    k, v = qkv[:, 32 * 128:40 * 128].view(5, 8, 128), qkv[:, 40 * 128:].view(5, 8, 128)
    ops.store_kvcache(k, v, c, c, torch.arange(5, dtype=torch.int32), ks, vs)
    (name, a), = rec.calls
    assert name == "nva_store_kvcache_fp8" and a[1] == a[3] == 48 * 128
    assert a[6:11] == (ks.data_ptr(), vs.data_ptr(), 4, 256, 32)
    assert a[12:15] == (5, 8, 128)


@pytest.mark.parametrize("bad", ["no scales", "one scale", "dtype", "scale shape", "scale dtype", "rows dtype", "heads",
                                 "bf16 cache", "slots"])
def test_store_refuses(rec, bad):
    from nvattn import ops
    c, (ks, vs) = cache()
    k = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    args = {
        "no scales": (k, k, c, c, slots),
        "one scale": (k, k, c, c, slots, ks),
        "dtype": (k, k, c.view(torch.float8_e5m2), c.view(torch.float8_e5m2), slots, ks, vs),
        "scale shape": (k, k, c, c, slots, ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()),
        "scale dtype": (k, k, c, c, slots, ks.half(), vs.half()),
        "rows dtype": (k.half(), k.half(), c, c, slots, ks, vs),
        "heads": (k[:, :4], k[:, :4], c, c, slots, ks, vs),
        "bf16 cache": (k, k, c.bfloat16(), c.bfloat16(), slots, ks, vs),
        "slots": (k, k, c, c, slots.long(), ks, vs),
    }[bad]
    with pytest.raises(AssertionError):
        ops.store_kvcache(*args)
    assert rec.calls == []


def test_decode_and_varlen_marshal(rec):
    from nvattn import ops
    c, (ks, vs) = cache()
    q = torch.zeros(3, 2, 32, 128, dtype=torch.bfloat16)
    lens, bt = torch.ones(3, dtype=torch.int32), torch.zeros(3, 7, dtype=torch.int32)[:, :5]
    out = ops.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens, block_table=bt, softmax_scale=0.1, k_scale=ks,
                                      v_scale=vs)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    ops.flash_attn_varlen_func(q.view(6, 32, 128), c, c, 4, cu, 9, cu, 0.1, block_table=bt[:2], k_scale=ks, v_scale=vs)
    (d, a), (w, b) = rec.calls
    assert d == "nva_paged_decode_fp8" and a[6:9] == (4, 256, 16) and a[11:18] == (7, 5, 3, 2, 32, 8, 128)
    assert w == "nva_varlen_attention_fp8" and b[6:9] == (4, 256, 16) and b[11:14] == (2, 6, 4) and b[15:17] == (7, 5)


@pytest.mark.parametrize("bad", ["no table", "group", "out", "lens", "head_dim", "not causal"])
def test_attention_refuses(rec, bad):
    from nvattn import _lib, ops
    c, (ks, vs) = cache(KVH=8)
    q = torch.zeros(3, 2, 32, 128, dtype=torch.bfloat16)
    lens, bt = torch.ones(3, dtype=torch.int32), torch.zeros(3, 5, dtype=torch.int32)
    cu = torch.tensor([0, 2, 4, 6], dtype=torch.int32)
    kw = dict(softmax_scale=0.1, k_scale=ks, v_scale=vs)
    with pytest.raises((AssertionError, _lib.NvattnError)):
        if bad == "no table":
            ops.flash_attn_varlen_func(q.view(6, 32, 128), c, c, 2, cu, 9, cu, 0.1, k_scale=ks, v_scale=vs)
        elif bad == "group":
            one, (k1, v1) = cache(KVH=1)
            ops.flash_attn_with_kvcache(torch.zeros(3, 1, 41, 128, dtype=torch.bfloat16), one, one, cache_seqlens=lens,
                                        block_table=bt, softmax_scale=0.1, k_scale=k1, v_scale=v1)
        elif bad == "out":
            ops.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens, block_table=bt, out=torch.zeros(3, 2, 32, 128), **kw)
        elif bad == "lens":
            ops.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens.long(), block_table=bt, **kw)
        elif bad == "head_dim":
            ops.flash_attn_with_kvcache(torch.zeros(3, 2, 32, 64, dtype=torch.bfloat16), c, c, cache_seqlens=lens,
                                        block_table=bt, **kw)
        else:
            ops.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens, block_table=bt, causal=False, **kw)
    assert rec.calls == []


def test_sampler_marshals_and_refuses(rec):
    from nvattn import sampler
    x = torch.zeros(3, 11)
    t, u = torch.ones(3), torch.zeros(3, dtype=torch.float64)
    ids = sampler.sample_tokens(x, t, u, top_k=torch.zeros(3, dtype=torch.int32))
    (name, a), = rec.calls
    assert name == "nva_sample_tokens" and a[1:5] == (11, 3, 11, 4) and a[7] == a[8] == 0 and a[10] == 8
    assert ids.shape == (3,) and ids.dtype == torch.int64
    for bad in (dict(temperatures=t[:2]), dict(uniforms=u.half()), dict(top_k=torch.zeros(3)), dict(top_p=u),
                dict(min_p=t[:1]), dict(logits=x.half()), dict(logits=x.t())):
        kw = {**dict(logits=x, temperatures=t, uniforms=u), **bad}
        with pytest.raises(AssertionError):
            sampler.sample_tokens(**kw)
    with pytest.raises(AssertionError):    # rows of logits and sequences do not go together
        sampler.verify_drafts_sampled(x, torch.zeros(3, 2, dtype=torch.int64), torch.ones(3, dtype=torch.int64), t,
                                      torch.zeros(3, 2, dtype=torch.float64), u)
    with pytest.raises(AssertionError):    # one uniforms' dtype for both
        sampler.verify_drafts_sampled(torch.zeros(9, 11), torch.zeros(3, 2, dtype=torch.int64),
                                      torch.ones(3, dtype=torch.int64), t, torch.zeros(3, 2), u)


def test_ops_refuse_cpu_tensors():
    from nvattn import ops, sampler
    c, (ks, vs) = cache()
    k = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.store_kvcache(k, k, c, c, torch.zeros(1, dtype=torch.int32), ks, vs)
    with pytest.raises(ValueError, match="CUDA"):
        sampler.sample_tokens(torch.zeros(2, 5), torch.ones(2), torch.zeros(2))


# ---------------------------------------------------------------------------------------------- the C ABI
def test_entry_points_refuse_on_the_host():
    from nvattn import _lib
    lib = _lib.load()
    store = [16, 1024, 16, 1024, 16, 16, 16, 16, 4, 256, 16, 16, 5, 8, 128, 0]

    def with_(args, **at):
        return [at.get("a%d" % i, v) for i, v in enumerate(args)]

    f = lib.nva_store_kvcache_fp8
    assert f(*with_(store, a12=0)) == 0                                             # no tokens: nothing to do
    assert f(*with_(store, a12=-1)) == 1 and f(*with_(store, a1=1000)) == 1 and f(*with_(store, a0=0)) == 1
    assert f(*with_(store, a14=64)) == 2                                            # head_dim
    for g in (4, 12, 512):
        assert f(*with_(store, a10=g)) == 2
    assert f(*with_(store, a9=264)) == 2 and f(*with_(store, a8=1 << 24)) == 2      # block size, slots past 31 bits
    assert f(*with_(store, a0=4)) == 3 and f(*with_(store, a1=1026)) == 3
    dec = [16, 4096, 16, 16, 16, 16, 4, 256, 16, 16, 16, 5, 5, 3, 1, 32, 8, 128, 0.1, 16, 4096, 16, 1 << 30, 0]
    f = lib.nva_paged_decode_fp8
    assert f(*with_(dec, a13=0)) == 0
    assert f(*with_(dec, a14=0)) == 1 and f(*with_(dec, a15=30)) == 1 and f(*with_(dec, a12=6)) == 1
    for bad in (0.0, -1.0, math.nan, math.inf):
        assert f(*with_(dec, a18=bad)) == 1
    assert f(*with_(dec, a17=64)) == 2 and f(*with_(dec, a7=192)) == 2 and f(*with_(dec, a8=24)) == 2
    assert f(*with_(dec, a15=41 * 8, a1=41 * 8 * 128, a20=41 * 8 * 128)) == 2       # 41 q heads per kv head
    assert f(*with_(dec, a0=8)) == 3 and f(*with_(dec, a1=4100)) == 3
    var = [16, 4096, 16, 16, 16, 16, 4, 256, 16, 16, 16, 3, 9, 4, 16, 5, 5, 32, 8, 128, 0.1, 16, 4096, 16, 1 << 30, 0]
    f = lib.nva_varlen_attention_fp8
    assert f(*with_(var, a12=0)) == 0 and f(*with_(var, a13=-1)) == 1 and f(*with_(var, a9=0)) == 1
    assert f(*with_(var, a20=math.nan)) == 1 and f(*with_(var, a19=64)) == 2
    smp = [16, 100, 3, 100, 4, 16, 0, 0, 0, 16, 4, 16, 16, 1 << 20, 0]
    f = lib.nva_sample_tokens
    assert f(*with_(smp, a2=0)) == 0
    assert f(*with_(smp, a1=99)) == 1 and f(*with_(smp, a5=0)) == 1 and f(*with_(smp, a3=0)) == 1
    assert f(*with_(smp, a4=8)) == 2 and f(*with_(smp, a10=2)) == 2
    assert f(*with_(smp, a3=400000, a1=400000)) == 2 and f(*with_(smp, a2=(1 << 20) + 1)) == 2
    assert f(*with_(smp, a0=18)) == 3 and f(*with_(smp, a11=4)) == 3
    assert f(*with_(smp, a12=0)) == 4 and f(*with_(smp, a13=3 * 32 - 1)) == 4 and f(*with_(smp, a12=8)) == 4
    ver = [16, 100, 3, 2, 100, 4, 16, 2, 16, 8, 16, 0, 0, 0, 16, 2, 16, 4, 16, 16, 16, 9 * 32, 0]
    f = lib.nva_verify_sampled
    assert f(*with_(ver, a2=0)) == 0
    assert f(*with_(ver, a3=-1)) == 1 and f(*with_(ver, a7=1)) == 1 and f(*with_(ver, a14=0)) == 1
    assert f(*with_(ver, a9=2)) == 2 and f(*with_(ver, a21=9 * 32 - 1)) == 4 and f(*with_(ver, a20=0)) == 4
    assert lib.nva_sample_workspace_bytes(9, 100, 4) == 9 * 32 and lib.nva_sample_workspace_bytes(1, 2049, 2) == 48


# ---------------------------------------------------------------------------------------------- restatements
def test_e4m3_restatement_is_torchs():
    x = torch.cat([torch.arange(-448, 449).double(), torch.randn(4000, dtype=torch.float64) * 20,
                   torch.randn(4000, dtype=torch.float64) * 2.0 ** -8, torch.exp2(torch.arange(-14, 9).double()) * 1.0625])
    x = x.float().double()
    assert torch.equal(fp8_cache.e4m3(x).float(), x.float().clamp(-448, 448).to(torch.float8_e4m3fn).float())


def test_store_restatement_keeps_blocks_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    c = torch.zeros(2, 256, 2, 128, dtype=torch.float8_e4m3fn)
    s = torch.zeros(2, 2, 16)
    x = torch.randn(40, 2, 128, generator=g).bfloat16() * torch.exp2(torch.randint(-3, 4, (40, 1, 1), generator=g))
    for i in range(40):    # token by token, as decoding does
        fp8_cache.store_ref(x[i:i + 1], c, s, torch.tensor([i]))
    got = fp8_cache.values(c, s)[0, :40]
    step = s.double().transpose(1, 2).repeat_interleave(16, dim=1)[0, :40, :, None]
    # one rounding to the block's last scale and at most one per growth before it, each half a step (2^-4 relative or
    # 2^-10 of the scale); a growth doubles the scale at least, so steps add up to less than twice the last one
    assert ((got - x.double()).abs() <= 2 * (2.0 ** -4 * x.double().abs() + 2.0 ** -10 * step)).all()


@pytest.mark.parametrize("settings", [{}, {"top_k": 3}, {"top_p": 0.7}, {"min_p": 0.2}, {"top_k": 4, "top_p": 0.6}])
def test_speculative_sampling_draws_the_target_distribution(settings):
    """Enumerated over a grid of both uniform numbers: accepted draft or redraw together give the row's weights."""
    rng = np.random.default_rng(3)
    logits = rng.normal(size=(2, 7)) * 1.5
    p = sampling.kept_weights(logits[0], 0.8, **settings)
    p = p / p.sum()
    N = 400
    grid = (np.arange(N) + 0.5) / N
    for d in range(7):
        count = np.zeros(7)
        accepted = sum(sampling.verify(logits, [d], 1, 0.8, [a], 0.5, **settings)[0] for a in grid) / N
        for u in grid:
            a, nxt = sampling.verify(logits, [d], 1, 0.8, [0.999999], u, **settings)
            if a == 0:
                count[nxt] += 1 / N
        total = (1 - accepted) * count
        total[d] += accepted
        # (a grid of N points is off by at most 1 / N per boundary)
        assert np.abs(total - p).max() <= 2 / N + 1e-12 or p[d] > 0.999


def test_three_parts_of_a_weight():
    """The 8-bit attention kernels' weights, bit by bit: float16, then three times the nearest number of three
    significant bits (the upper byte, an e5m2 value) and the rest.  float16 loses 2^-11 of the weight at most (2^-25 of
    subnormal ones), the parts half their smallest step, 2^-17."""
    w = np.concatenate([np.exp2(np.random.default_rng(0).uniform(-30, 15, 200000)), np.exp2(np.arange(-30, 16.0)),
                        np.float16(np.arange(0x7801, dtype=np.uint16).view(np.float16)).astype(np.float64)])
    w = w.astype(np.float32)
    x = w.astype(np.float16)
    total = np.zeros_like(w, dtype=np.float64)
    for part in range(3):
        bits = x.view(np.uint16).astype(np.uint32) + 0x80
        assert (bits < 0x10000).all()
        y = (bits & 0xFF00).astype(np.uint16).view(np.float16)
        e5m2 = torch.from_numpy((bits >> 8).astype(np.uint8)).view(torch.float8_e5m2).double().numpy()
        assert np.array_equal(e5m2, y.astype(np.float64))
        rest = x.astype(np.float64) - e5m2
        assert np.array_equal(rest, (x - y).astype(np.float64))
        total += e5m2
        x = x - y
    assert (np.abs(total - w) <= np.maximum(2.0 ** -11 * w, 2.0 ** -25) + 2.0 ** -17).all()


# ---------------------------------------------------------------------------------------------- rows that overlap
@pytest.fixture()
def checked(rec, monkeypatch):
    """The wrappers with the library's own argument checks behind them (the size queries alone, which ask for the
    device, are answered here)."""
    from nvattn import _lib
    real = ctypes.CDLL(_lib.LIB_PATH)
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(real, name)
        fn.restype, fn.argtypes = res, args

    class Checked:
        nva_paged_attention_fp8_workspace_bytes = staticmethod(rec.nva_paged_attention_fp8_workspace_bytes)
        nva_sample_workspace_bytes = staticmethod(rec.nva_sample_workspace_bytes)

        def __getattr__(self, name):
            return getattr(real, name)

    monkeypatch.setattr(_lib, "load", lambda: Checked())


@pytest.mark.parametrize("what", ["block table", "varlen block table", "logits", "sample logits", "drafts", "one draft",
                                  "accept uniforms"])
def test_expanded_views_are_refused(checked, what):
    """Rows that share memory have a stride of 0, which no call may take for a row's width: it would read past them."""
    from nvattn import _lib, ops
    c, (ks, vs) = cache()
    q = torch.zeros(3, 2, 32, 128, dtype=torch.bfloat16)
    lens, cu = torch.ones(3, dtype=torch.int32), torch.tensor([0, 2, 4, 6], dtype=torch.int32)
    table = torch.zeros(1, 5, dtype=torch.int32).expand(3, -1)
    S, K, V = 3, 1 if what == "one draft" else 2, 11
    kw = dict(logits=torch.zeros(S * (K + 1), V), draft_ids=torch.zeros(S, K, dtype=torch.int64),
              num_drafts=torch.ones(S, dtype=torch.int64), temperatures=torch.ones(S),
              accept_uniforms=torch.zeros(S, K), uniforms=torch.zeros(S))
    with pytest.raises(_lib.NvattnError, match="invalid argument"):
        if what == "block table":
            ops.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens, block_table=table, softmax_scale=0.1, k_scale=ks,
                                        v_scale=vs)
        elif what == "varlen block table":
            ops.flash_attn_varlen_func(q.view(6, 32, 128), c, c, 2, cu, 9, cu, 0.1, block_table=table, k_scale=ks,
                                       v_scale=vs)
        elif what == "sample logits":
            ops.sample_tokens(torch.zeros(1, V).expand(S, V), torch.ones(S), torch.zeros(S))
        else:
            name = {"logits": "logits", "drafts": "draft_ids", "one draft": "draft_ids",
                    "accept uniforms": "accept_uniforms"}[what]
            kw[name] = kw[name][:1].expand(kw[name].shape)
            ops.verify_sampled(**kw)


def test_single_rows_need_no_stride(rec):
    """One sequence: its rows' stride says nothing, also where a view makes it 0."""
    from nvattn import ops
    c, (ks, vs) = cache()
    table = torch.zeros(5, dtype=torch.int32).as_strided((1, 5), (0, 1))
    ops.flash_attn_with_kvcache(torch.zeros(1, 2, 32, 128, dtype=torch.bfloat16), c, c,
                                cache_seqlens=torch.ones(1, dtype=torch.int32), block_table=table, softmax_scale=0.1,
                                k_scale=ks, v_scale=vs)
    ops.sample_tokens(torch.zeros(11).as_strided((1, 11), (0, 1)), torch.ones(1), torch.zeros(1))
    ops.verify_sampled(torch.zeros(3, 11), torch.zeros(2, dtype=torch.int64).as_strided((1, 2), (0, 1)),
                       torch.ones(1, dtype=torch.int64), torch.ones(1), torch.zeros(2).as_strided((1, 2), (0, 1)),
                       torch.zeros(1))
    (_, a), (_, s), (_, v) = rec.calls
    assert a[11:13] == (5, 5) and s[1] == 11 and v[1] == 11 and v[7] == 2 and v[15] == 2
