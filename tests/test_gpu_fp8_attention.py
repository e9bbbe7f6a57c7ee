"""Attention over an 8-bit cache against float64 over the values the cache stands for.  Tolerances are the bound of
oracle.fp8_cache.attention_ref, element by element."""
import pytest
import torch

from oracle import fp8_cache

pytestmark = pytest.mark.gpu


def make(lens, H=32, KVH=8, G=16, qlens=None, n=1, seed=0, spread=0, size=1.0, spare=3, BS=256):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages_of = [(x + BS - 1) // BS for x in lens]
    NB = sum(pages_of) + spare
    x = torch.randn(2, NB, BS // G, G, KVH, 128, generator=g, device="cuda") * size
    if spread:    # blocks of very different magnitude
        x *= torch.exp2(torch.randint(-spread, spread + 1, (2, NB, BS // G, 1, KVH, 1), generator=g, device="cuda"))
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(3, 5)) / 448)))
    c = (x / s[:, :, :, None, :, None]).to(torch.float8_e4m3fn).view(2, NB, BS, KVH, 128)
    s = s.transpose(2, 3).contiguous()
    order = torch.randperm(NB, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(1, max(pages_of))), -1, dtype=torch.int32)
    at = 0
    for b, w in enumerate(pages_of):
        table[b, :w] = torch.tensor(order[at:at + w], dtype=torch.int32)
        at += w
    T = sum(qlens) if qlens is not None else len(lens) * n
    q = torch.randn(T, H, 128, generator=g, device="cuda").bfloat16()
    cu = lambda xs: torch.tensor([0] + list(xs)).cumsum(0).int().cuda()  # noqa: E731
    return dict(q=q if qlens is not None else q.view(len(lens), n, H, 128), c=(c[0], c[1]), s=(s[0], s[1]),
                lens=list(lens), table=table.cuda(),
                lens_d=torch.tensor(lens, dtype=torch.int32, device="cuda"), n=n, qlens=qlens,
                cu_q=cu(qlens) if qlens is not None else None, cu_k=cu(lens), scale=128 ** -0.5)


def run(b, out=None, max_q=None):
    from nvattn import ops
    if b["qlens"] is not None:
        return ops.flash_attn_varlen_func(b["q"], b["c"][0], b["c"][1], max_seqlen_q=max_q or max(b["qlens"]),
                                          cu_seqlens_q=b["cu_q"], max_seqlen_k=max(b["lens"]), cu_seqlens_k=b["cu_k"],
                                          softmax_scale=b["scale"], causal=True, block_table=b["table"], out=out,
                                          k_scale=b["s"][0], v_scale=b["s"][1])
    return ops.flash_attn_with_kvcache(b["q"], b["c"][0], b["c"][1],
                                       cache_seqlens=b["lens_d"],
                                       block_table=b["table"], softmax_scale=b["scale"], out=out, k_scale=b["s"][0],
                                       v_scale=b["s"][1])


def ref(b):
    starts = b["cu_q"].tolist() if b["qlens"] is not None else None
    return fp8_cache.paged_ref(b["q"], b["c"], b["s"], b["lens"], b["table"], b["scale"], starts)


def check(b, got=None, what=""):
    from nvattn import _lib
    got = run(b) if got is None else got
    want, bound = ref(b)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.2f} times the bound, off {float(off.max()):.3g}"
    assert _lib.device_error() == 0
    return got


@pytest.mark.parametrize("lens", [[1], [15], [16], [17], [127], [128], [129], [255], [256], [257], [385],
                                  [1, 2, 3, 300, 511, 512, 513, 1000]])
def test_decode_lengths(cuda, lens):
    check(make(lens, seed=lens[0]))


@pytest.mark.parametrize("H,KVH", [(16, 8), (8, 1), (40, 8), (4, 4), (7, 1), (40, 1), (12, 6), (64, 16)])
@pytest.mark.parametrize("G", [8, 256])
def test_head_layouts(cuda, H, KVH, G):
    check(make([300, 77, 1500], H=H, KVH=KVH, G=G, seed=H))


@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 10, 11, 17, 40])
def test_several_queries(cuda, n):
    """Every row width of the kernel, and runs longer than one piece of 40 rows."""
    check(make([n, 200, 256, 257, 1024, 1500], n=n, G=32, seed=n))


@pytest.mark.parametrize("lens", [[9], [127], [128, 136], [137, 263], [264, 265], [383, 384, 385]])
def test_query_runs_at_tile_edges(cuda, lens):
    check(make(lens, n=9, G=128, seed=lens[0]))


def test_split_long_sequence(cuda):
    check(make([9000], seed=3))
    check(make([20000, 5], KVH=1, H=4, seed=4))


def test_blocks_of_very_different_scale(cuda):
    check(make([700, 1300, 129], spread=12, size=2.0 ** -6, seed=5, G=16), what="spread")


def test_a_token_far_above_a_long_tail(cuda):
    """One token 13 (natural units) above 60,000 equal ones: their weights are e^-13 of its, and together a tenth."""
    L = 60000
    b = make([L], H=4, KVH=1, seed=6)
    k, v = b["c"]
    k.view(torch.uint8).zero_()
    b["s"][0].fill_(2.0 ** -4)
    b["q"].zero_()
    b["q"][..., 0] = 128 ** 0.5 * 13 / 16
    first = int(b["table"][0, 0])
    k.view(torch.float8_e4m3fn)[first, 0, 0, 0] = 256.0        # 256 * 2^-4 = 16: a score of 13
    got = check(b)
    assert float(got.float().abs().max()) > 0


def test_padding_sequences_and_poison_behind_the_context(cuda):
    from nvattn import _lib
    lens = [130, 0, 77, 300, 0]
    b = make(lens, seed=7)
    want, bound = ref(b)
    for c, s in zip(b["c"], b["s"]):
        raw = c.view(torch.uint8)
        for i, L in enumerate(lens):
            for col in range(b["table"].shape[1]):
                page = int(b["table"][i, col])
                if page < 0:
                    continue
                for p in range(256):
                    if col * 256 + p >= L:
                        raw[page, p] = 0x7F                       # NaN
                last = max(0, min(16, (L - col * 256 + 15) // 16))
                s[page, :, last:] = float("nan")
    got = run(b)
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all()
    assert (got[1] == 0).all() and (got[4] == 0).all() and _lib.device_error() == 0


@pytest.mark.parametrize("qlens", [[81, 200, 300, 1], [80, 129, 17, 82]])
def test_long_runs_with_poison_behind_the_context(cuda, qlens):
    """Runs on either side of the length from which a kernel of their own takes them, pages full of NaN past the keys."""
    from nvattn import _lib
    lens = [81, 456, 300, 90]
    b = make(lens, qlens=qlens, seed=23, spread=6, size=0.1)
    want, bound = ref(b)
    for c, s in zip(b["c"], b["s"]):
        raw = c.view(torch.uint8)
        for i, L in enumerate(lens):
            for col in range((L + 255) // 256):
                page = int(b["table"][i, col])
                raw[page, max(0, L - col * 256):] = 0xFF
                last = max(0, min(16, (L - col * 256 + 15) // 16))
                s[page, :, last:] = float("inf")
    got = run(b)
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all() and _lib.device_error() == 0


def test_long_run_without_keys_and_bad_pages(cuda):
    from nvattn import _lib
    b = make([0, 50, 700], qlens=[130, 200, 90], seed=24)
    got = check(b)
    assert (got[:130] == 0).all() and (got[130:280] == 0).all()
    b["table"][2, 1] = -7
    got = run(b)
    assert torch.isfinite(got).all() and _lib.device_error() & 4
    _lib.clear_device_error()


def test_rows_without_a_key(cuda):
    """More queries than keys: the first rows see nothing and are zero, in pieces with and without keys."""
    b = make([3, 30, 12], n=20, seed=8)
    got = check(b)
    assert (got[0, :17] == 0).all() and (got[2, :8] == 0).all()


@pytest.mark.parametrize("qlens,lens", [([1], [1]), ([200, 1, 300], [456, 90, 300]), ([0, 5, 0, 1], [40, 5, 0, 700]),
                                        ([13, 1, 1, 64, 2], [13, 500, 1, 900, 131]), ([1000], [1000]),
                                        ([7, 50], [3, 20]), ([4, 4, 4], [0, 4, 0]), ([40, 1, 8, 16, 9], [40, 1, 8, 16, 9]),
                                        ([33] * 5 + [1] * 70, [900] * 5 + list(range(1, 1400, 20))),
                                        ([2500], [5000])])
def test_varlen(cuda, qlens, lens):
    check(make(lens, qlens=qlens, seed=sum(qlens)))


@pytest.mark.parametrize("H,KVH", [(8, 1), (16, 8), (20, 4), (40, 1), (33, 1), (32, 1), (4, 4), (14, 2)])
def test_varlen_head_layouts(cuda, H, KVH):
    check(make([300, 77, 520, 33], H=H, KVH=KVH, qlens=[100, 1, 9, 33], seed=H, G=64))


@pytest.mark.parametrize("qlens", [[1] * 8 + [60] * 2, [60] * 2 + [1] * 96, [20] * 16, [5] * 64, [63] * 3, [64] * 3,
                                   [9] * 16 + [1] * 130, [1, 63, 1, 5, 64, 1, 17], [33] * 5, [7] * 2 + [1] * 200])
@pytest.mark.parametrize("H", [32, 8])
def test_varlen_kernel_choice(cuda, qlens, H):
    """Both sides of the bounds at which runs go to another kernel."""
    lens = [n + (37 * i) % 300 for i, n in enumerate(qlens)]
    lens[1] = max(qlens[1] - 3, 0)                         # keys for some of its queries only
    check(make(lens, H=H, qlens=qlens, seed=len(qlens) + H))


def test_varlen_rows_behind_the_last_sequence_stay(cuda):
    b = make([300, 50], qlens=[100, 1], seed=9)
    big = torch.cat([b["q"], b["q"][:20]])
    out = torch.full_like(big, 7.0)
    b2 = dict(b, q=big)
    run(b2, out=out)
    check(b, got=out[:101])
    assert (out[101:] == 7).all()


def test_varlen_bound_below_the_longest_run(cuda):
    """max_seqlen_q only picks the row width: longer runs are still whole."""
    b = make([300, 77], qlens=[90, 3], seed=10)
    check(b, got=run(b, max_q=1))


def test_many_sequences(cuda):
    """More sequences than a block of the work split scans at once."""
    g = torch.Generator().manual_seed(0)
    check(make(torch.randint(0, 200, (700,), generator=g).tolist(), H=8, KVH=2, seed=11))
    lens = torch.randint(1, 60, (600,), generator=g).tolist()
    check(make(lens, H=4, KVH=1, qlens=[min(x, 1 + i % 5) for i, x in enumerate(lens)], seed=12))


def test_queries_that_are_no_numbers_stay_in_their_rows(cuda):
    b = make([300, 200], n=2, seed=13)
    want, bound = ref(b)
    b["q"][1, 0, 5, 3] = float("nan")
    b["q"][0, 1, 9, 0] = float("inf")
    got = run(b)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[1, 0, 5] = bad[0, 1, 9] = True
    assert torch.isnan(got[bad]).all()
    assert ((got.double() - want).abs() <= bound)[~bad].all()


def test_bad_pages_are_flagged_and_read_nothing(cuda):
    from nvattn import _lib
    _lib.clear_device_error()
    b = make([300, 200], seed=14)
    b["table"][0, 1] = b["c"][0].shape[0] + 5
    got = run(b)
    torch.cuda.synchronize()
    assert _lib.device_error() & 4 and torch.isfinite(got).all()
    _lib.clear_device_error()
    want, bound = ref(make([300, 200], seed=14))
    assert ((got.double() - want).abs() <= bound)[1].all()
    b = make([300], seed=15)
    b["table"] = b["table"][:, :1]                                # a table too narrow for the context
    assert torch.isfinite(run(b)).all() and _lib.device_error() & 4
    _lib.clear_device_error()


def test_strided_queries_and_output(cuda):
    b = make([300, 77, 513], n=2, seed=16)
    wide = torch.zeros(6, 48 * 128, dtype=torch.bfloat16, device="cuda")
    wide[:, :32 * 128] = b["q"].reshape(6, -1)
    out = torch.full((6, 40 * 128), 5.0, dtype=torch.bfloat16, device="cuda")
    view = out[:, :32 * 128].view(3, 2, 32, 128)
    run(dict(b, q=wide[:, :32 * 128].view(3, 2, 32, 128)), out=view)
    check(b, got=view)
    assert (out[:, 32 * 128:] == 5).all()


def test_a_cache_past_four_gigabytes(cuda):
    """Pages whose bytes start past 2^32 and whose rows lie past 2^24."""
    b = make([700, 300], seed=17, spare=2)
    NB = 17000
    far = torch.arange(NB - b["c"][0].shape[0], NB, device="cuda")
    c2 = [torch.empty(NB, 256, 8, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s2 = [torch.ones(NB, 8, 16, device="cuda") for _ in range(2)]
    for i in range(2):
        c2[i][far] = b["c"][i].view(torch.uint8)
        s2[i][far] = b["s"][i]
    got = run(dict(b, c=[x.view(torch.float8_e4m3fn) for x in c2], s=s2,
                   table=torch.where(b["table"] < 0, b["table"], b["table"] + int(far[0]))))
    check(b, got=got)


def test_one_workspace_serves_both_caches_and_graphs(cuda):
    """8-bit and bf16 calls in turn, eager and replayed, share the merge tickets: same bits every time."""
    from nvattn import ops
    b = make([4000, 300, 1900], seed=18)
    v = make([300, 600], qlens=[150, 1], seed=19)
    kc = [x.bfloat16() for x in b["c"]]
    ops.reserve_workspace(64, 4096, 32, 8, fp8_cache=True)

    def calls():
        return (run(b), run(v), ops.flash_attn_with_kvcache(b["q"], kc[0], kc[1], cache_seqlens=b["lens_d"],
                                                            block_table=b["table"], softmax_scale=0.01))
    first = [x.clone() for x in calls()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls()
    side = torch.cuda.Stream()
    for i in range(20):
        if i % 3 == 0:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                again = calls()
            torch.cuda.current_stream().wait_stream(side)
        elif i % 3 == 1:
            again = calls()
        else:
            for x in held:
                x.zero_()
            graph.replay()
            again = held
        for x, y in zip(first, again):
            assert torch.equal(x, y)
    check(b, got=first[0])
    check(v, got=first[1])


def test_long_replays_stay_clean(cuda):
    from nvattn import _lib
    g = torch.Generator().manual_seed(1)
    b = make(torch.randint(16, 3000, (64,), generator=g).tolist(), seed=20)
    v = make([600, 900] + torch.randint(16, 2000, (60,), generator=g).tolist(), qlens=[600, 300] + [1] * 60, seed=21)
    k = make(torch.randint(16, 2000, (32,), generator=g).tolist(), n=9, seed=22)
    for case in (b, v, k):
        want = run(case)
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(case, out=out)
        for _ in range(100):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and _lib.device_error() == 0


def test_split_calls_in_a_row_and_replayed(cuda):
    """Calls whose kernels overlap share one workspace, back to back and in a graph: every output is the first one's."""
    from nvattn import _lib
    batches = [make([40 + (53 * i) % 900 for i in range(len(q))], qlens=q, seed=30 + i)
               for i, q in enumerate([[1] * 90 + [20] * 6, [1] * 70 + [5] * 9 + [130], [60] * 2 + [1] * 100, [9] * 40])]
    want = [check(b) for b in batches]
    outs = [torch.empty_like(w) for w in want]

    def step():
        for b, o in zip(batches, outs):
            run(b, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(60):
        for o in outs:
            o.fill_(7.0)
        graph.replay() if i % 2 else step()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), i
    assert _lib.device_error() == 0


@pytest.mark.parametrize("H", [16, 9, 40, 8])
def test_varlen_bound_of_zero(cuda, H):
    """A bound of 0 on runs that are there, with more q heads per kv head than the smallest tile has rows."""
    from nvattn import _lib, ops
    lib = _lib.load()
    assert lib.nva_paged_attention_fp8_workspace_bytes(0, H, 1, 128) == \
        lib.nva_paged_attention_fp8_workspace_bytes(1, H, 1, 128)
    b = make([300, 77, 5], H=H, KVH=1, qlens=[90, 3, 1], seed=40)
    check(b, got=ops.flash_attn_varlen_func(b["q"], *b["c"], max_seqlen_q=0, cu_seqlens_q=b["cu_q"], max_seqlen_k=300,
                                            cu_seqlens_k=b["cu_k"], softmax_scale=b["scale"], block_table=b["table"],
                                            k_scale=b["s"][0], v_scale=b["s"][1]))


@pytest.mark.parametrize("scale,taken", [(0.0, 2.0 ** -40), (2.0 ** -60, 2.0 ** -40), (float("nan"), 2.0 ** -40),
                                         (2.0 ** 50, 2.0 ** 40), (float("inf"), 2.0 ** 40)])
@pytest.mark.parametrize("qlen", [3, 63, 64, 200])
def test_v_scales_out_of_range(cuda, scale, taken, qlen):
    """They count as the bounds of the range, whichever kernel takes the run."""
    b = make([300], qlens=[qlen], seed=41)
    b["s"][1].fill_(taken)
    want, bound = ref(b)
    b["s"][1].fill_(scale)
    got = run(b)
    assert ((got.double() - want).abs() <= bound).all()


def far_token_and_tails(gaps, B, L, spread, seed, varlen=False):
    """B sequences of L tokens; in row i of each the first token's score lies gaps[i] above those of the others (apart
    from each other by `spread`), whose values are around 1 where the first one's are 0: the output is the tail's share."""
    n = len(gaps)
    b = make([L] * B, H=1, KVH=1, n=n, qlens=[n] * B if varlen else None, seed=seed)
    q = b["q"].view(B, n, 128)
    q.zero_()
    q[..., 0] = torch.tensor([g * 128 ** 0.5 / 16 for g in gaps])
    q[..., 1] = spread * 128 ** 0.5
    c = [x.view(torch.uint8).zero_().view(torch.float8_e4m3fn) for x in b["c"]]
    for s in b["s"]:
        s.fill_(2.0 ** -4)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c[0][..., 1] = (torch.randn(c[0].shape[:3], generator=g, device="cuda") * 16).to(torch.float8_e4m3fn)
    c[1].copy_((torch.rand(c[1].shape, generator=g, device="cuda") * 8 + 12).to(torch.float8_e4m3fn))
    for page in b["table"][:, 0].long().tolist():
        c[0].view(torch.uint8)[page, 0, 0, :2] = torch.tensor([0x78, 0], dtype=torch.uint8)    # 256 * 2^-4 = 16, 0
        c[1].view(torch.uint8)[page, 0, 0] = 0
    return dict(b, c=c)


@pytest.mark.parametrize("B,L,spread", [(300, 4000, 0.0), (300, 4000, 0.05), (300, 700, 1.0), (1, 60000, 0.0)])
@pytest.mark.parametrize("rows", [8, 16, 24, 32, 40, 80])
def test_the_tail_behind_a_far_token_keeps_its_weight(cuda, B, L, spread, rows):
    """Gaps that put the tail's weights at every place between two powers of two, by every kernel (80 rows: the prefill
    kernel's) and with few enough CTAs a sequence that one CTA has both.  The tail's weights are all rounded alike, so
    their errors add up; without the tail the output would be 0."""
    gaps = [4 + 11 * i / rows for i in range(rows)]
    b = far_token_and_tails(gaps, B, L, spread, seed=rows, varlen=rows == 80)
    want, bound = ref(b)
    assert (want > 20 * bound).all()
    check(b)


@pytest.mark.parametrize("n", [1, 4, 5, 10])
@pytest.mark.parametrize("far", [2.0 ** 6, 2.0 ** 11, 2.0 ** 15])
def test_queries_with_one_large_value(cuda, n, far):
    """q's two e4m3 parts hold values down to 2^-10 of their row's largest whole and are off by 2^-18 of it at most below
    (include/nvattn.h): scores by that times the sum of |k|, weights by twice as much of themselves."""
    b = make([700, 1300, n], n=n, seed=50 + n, size=0.3)
    b["c"][0].view(torch.uint8)[..., 7] = 0                     # (the large value meets no key: the small ones decide)
    b["q"][..., 7] = far
    want, bound = ref(b)
    size, _ = ref(dict(b, c=(b["c"][0], (b["c"][1].view(torch.uint8) & 0x7F).view(torch.float8_e4m3fn))))
    keys = fp8_cache.values(b["c"][0], b["s"][0]).abs().sum(-1).max()
    bound = bound + 2 * 2.0 ** -18 * far * keys * b["scale"] * size
    assert ((run(b).double() - want).abs() <= bound).all()
