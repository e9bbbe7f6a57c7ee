"""The rounding scatter into an 8-bit cache, bit for bit against the float64 restatement: every byte of the cache and
every scale, written or not."""
import pytest
import torch

from oracle import fp8_cache

pytestmark = pytest.mark.gpu


def filled(g, NB, KVH, G, BS=256):
    """A cache as earlier calls left it (values of about 0.5)."""
    x = torch.randn(NB, BS // G, G, KVH, 128, generator=g) * 0.5
    amax = x.abs().amax(dim=(2, 4))
    s = torch.exp2(torch.ceil(torch.log2(amax / 448)))
    c = (x / s[:, :, None, :, None]).to(torch.float8_e4m3fn).view(NB, BS, KVH, 128)
    return c, s.transpose(1, 2).contiguous()


def check(rows, slots, c0, s0, c1=None, s1=None, stream=None):
    """One call against the restatement, k and v with different rows and caches."""
    from nvattn import ops
    c1 = c0.clone() if c1 is None else c1
    s1 = s0.clone() if s1 is None else s1
    T, KVH, _ = rows.shape
    k, v = rows, (rows.flip(0) * 1.5).to(torch.bfloat16)
    dev = [t.cuda() for t in (c0, c1)]
    sc = [t.cuda() for t in (s0, s1)]
    qkv = torch.zeros(T, 4 * KVH * 128, dtype=torch.bfloat16, device="cuda")    # strided rows, as the projection's
    qkv[:, 2 * KVH * 128:3 * KVH * 128] = k.reshape(T, -1).cuda()
    qkv[:, 3 * KVH * 128:] = v.reshape(T, -1).cuda()
    kd = qkv[:, 2 * KVH * 128:3 * KVH * 128].view(T, KVH, 128)
    vd = qkv[:, 3 * KVH * 128:].view(T, KVH, 128)
    ops.store_kvcache(kd, vd, dev[0], dev[1], slots.cuda(), sc[0], sc[1])
    for x, c, s, dc, ds, name in ((k, c0, s0, dev[0], sc[0], "k"), (v, c1, s1, dev[1], sc[1], "v")):
        rc, rs = c.clone(), s.clone()
        fp8_cache.store_ref(x, rc, rs, slots)
        assert torch.equal(ds.cpu(), rs), f"{name} scales"
        assert torch.equal(dc.cpu().view(torch.uint8), rc.view(torch.uint8)), f"{name} values"


@pytest.mark.parametrize("T,KVH,G", [(1, 8, 16), (3, 1, 8), (64, 8, 16), (33, 2, 256), (130, 4, 64), (257, 8, 32),
                                     (1000, 2, 128)])
def test_runs_of_positions(cuda, T, KVH, G):
    """Sequences that go on anywhere in a block: parts of blocks, whole blocks, blocks begun afresh."""
    g = torch.Generator().manual_seed(T * 131 + G)
    NB = T // 256 + 8
    c, s = filled(g, NB, KVH, G)
    rows = (torch.randn(T, KVH, 128, generator=g) * (0.1 + 2 * torch.rand(T, 1, 1, generator=g))).bfloat16()
    start = 100
    page = torch.randperm(NB, generator=g)
    pos = start + torch.arange(T)
    slots = (page[pos // 256] * 256 + pos % 256).int()
    check(rows, slots, c, s)


def test_any_order_skipped_and_repeated_slots(cuda):
    """Slots in no order, -1 among them, and slots named several times (the last token wins)."""
    g = torch.Generator().manual_seed(5)
    c, s = filled(g, 6, 2, 16)
    T = 700
    slots = torch.randint(0, 6 * 256, (T,), generator=g).int()
    slots[::9] = -1
    slots[500:520] = slots[0:20]
    slots[3] = slots[690] = slots[100]
    check((torch.randn(T, 2, 128, generator=g) * 3).bfloat16(), slots, c, s)


@pytest.mark.parametrize("G", [8, 16, 128])
def test_token_by_token_growth(cuda, G):
    """Louder and louder tokens join a block one call at a time: the scale grows and what it holds is rounded again."""
    g = torch.Generator().manual_seed(G)
    from nvattn import ops
    c, s = filled(g, 1, 2, G)
    d, ds = c.cuda(), s.cuda()
    e, es = c.cuda(), s.cuda()
    for i in range(24):
        row = (torch.randn(1, 2, 128, generator=g) * 1.6 ** i * 0.01).bfloat16()
        slot = torch.tensor([3 + i], dtype=torch.int32)
        ops.store_kvcache(row.cuda(), row.cuda(), d, e, slot.cuda(), ds, es)
        fp8_cache.store_ref(row, c, s, slot)
    assert torch.equal(ds.cpu(), s) and torch.equal(es.cpu(), s)
    assert torch.equal(d.cpu().view(torch.uint8), c.view(torch.uint8))


def test_zeros_tiny_huge_and_no_numbers(cuda):
    g = torch.Generator().manual_seed(1)
    c, s = filled(g, 2, 2, 16)
    rows = torch.randn(96, 2, 128, generator=g).bfloat16()
    rows[0:16] = 0                               # a block of zeros: the least scale
    rows[16:32] *= 2.0 ** -60                    # below the least scale's steps
    rows[32:48] *= 2.0 ** 90                     # past the largest scale: clamped
    rows[50, :, 3] = float("inf")                # NaN in the cache, without a say in the scale
    rows[51, 0, 7] = float("nan")
    rows[64:80, 1] = float("nan")                # nothing but NaN
    check(rows, torch.arange(96).int(), c, s)


def test_fresh_scales_of_zero(cuda):
    """Scales as kvcache_scales makes them, first write in the middle of a block (a prefix that was never stored)."""
    g = torch.Generator().manual_seed(2)
    c = torch.zeros(2, 256, 4, 128, dtype=torch.float8_e4m3fn)
    check(torch.randn(20, 4, 128, generator=g).bfloat16(), (torch.arange(20) + 7).int(), c, torch.zeros(2, 4, 16))


def test_out_of_range_slots_are_skipped_and_flagged(cuda):
    from nvattn import _lib, ops
    _lib.clear_device_error()
    g = torch.Generator().manual_seed(3)
    c, s = filled(g, 1, 2, 16)
    d, ds = c.cuda(), s.cuda()
    rows = torch.randn(3, 2, 128, generator=g).bfloat16()
    slots = torch.tensor([256, 5, -2], dtype=torch.int32)
    ops.store_kvcache(rows.cuda(), rows.cuda(), d, d.clone(), slots.cuda(), ds, ds.clone())
    assert _lib.device_error() & 1
    _lib.clear_device_error()
    fp8_cache.store_ref(rows[1:2], c, s, slots[1:2])
    assert torch.equal(d.cpu().view(torch.uint8), c.view(torch.uint8)) and torch.equal(ds.cpu(), s)


def test_no_tokens(cuda):
    from nvattn import ops
    c = torch.zeros(1, 256, 2, 128, dtype=torch.float8_e4m3fn, device="cuda")
    ks, vs = ops.kvcache_scales(c)
    x = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    ops.store_kvcache(x, x, c, c, torch.zeros(0, dtype=torch.int32, device="cuda"), ks, vs)


def test_replayed_graph_on_another_stream(cuda):
    from nvattn import ops
    g = torch.Generator().manual_seed(4)
    c, s = filled(g, 4, 8, 16)
    d, e, ds, es = c.cuda(), c.cuda(), s.cuda(), s.cuda()
    rows = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(4, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.store_kvcache(rows, rows, d, e, slots, ds, es)
        for i in range(5):
            x = torch.randn(4, 8, 128, generator=g).bfloat16() * (i + 1)
            at = torch.randperm(1024, generator=g)[:4].int()
            rows.copy_(x)
            slots.copy_(at)
            graph.replay()
            fp8_cache.store_ref(x, c, s, at)
    side.synchronize()
    assert torch.equal(d.cpu().view(torch.uint8), c.view(torch.uint8)) and torch.equal(es.cpu(), s)
