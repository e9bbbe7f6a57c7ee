"""Sampling and speculative sampling against the float64 restatement, token for token.  A draw whose uniform number lies
within 1e-9 of a boundary between tokens (relative to the sum) may go either way in float64 itself; the cases are made
with fixed seeds and none of them does (asserted)."""
import numpy as np
import pytest
import torch

from oracle import sampling

pytestmark = pytest.mark.gpu


def rows(R, V, dtype, seed, size=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * size
    return x.to(dtype), g


def run(x, t, u, **kw):
    from nvattn.sampler import sample_tokens
    dev = {k: v.cuda() for k, v in kw.items() if v is not None}
    return sample_tokens(x.cuda() if not x.is_cuda else x, t.cuda(), u.cuda(), **dev).cpu()


def check(x, t, u, top_k=None, top_p=None, min_p=None, got=None):
    R = x.shape[0]
    got = run(x, t, u, top_k=top_k, top_p=top_p, min_p=min_p) if got is None else got
    host = x.float().cpu().numpy()
    for r in range(R):
        want, margin = sampling.sample(host[r], float(t[r]), float(u[r]),
                                       int(top_k[r]) if top_k is not None else 0,
                                       float(top_p[r]) if top_p is not None else 1.0,
                                       float(min_p[r]) if min_p is not None else 0.0)
        assert margin > 1e-9 or got[r] == want, "the case itself is undecided"
        assert int(got[r]) == want, (r, int(got[r]), want)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 31, 33, 255, 1000, 4097, 32003])
def test_vocabularies(cuda, V, dtype):
    R = 12
    x, g = rows(R, V, dtype, V)
    u = torch.rand(R, generator=g)
    t = torch.rand(R, generator=g) * 1.5 + 0.2
    check(x, t, u)
    check(x, t, u, top_k=torch.randint(0, max(V, 2), (R,), generator=g).int())
    check(x, t, u, top_p=torch.rand(R, generator=g))
    check(x, t, u, min_p=torch.rand(R, generator=g) * 0.3)
    t[::3] = 0
    check(x, t, u.double(), top_k=torch.randint(0, 60, (R,), generator=g).int(), top_p=torch.rand(R, generator=g),
          min_p=torch.rand(R, generator=g) * 0.05)


@pytest.mark.parametrize("R,dtype", [(1, torch.bfloat16), (5, torch.float32), (40, torch.bfloat16)])
def test_a_whole_vocabulary(cuda, R, dtype):
    x, g = rows(R, 151936, dtype, R)
    u = torch.rand(R, generator=g, dtype=torch.float64)
    t = torch.rand(R, generator=g) + 0.4
    check(x, t, u)
    check(x, t, u, top_p=torch.full((R,), 0.97), top_k=torch.randint(0, 5000, (R,), generator=g).int())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_any_alignment_and_row_stride(cuda, dtype):
    base = torch.randn(9, 5003, generator=torch.Generator().manual_seed(1)).to(dtype).cuda() * 2
    g = torch.Generator().manual_seed(2)
    u, t = torch.rand(9, generator=g), torch.ones(9)
    for lo, hi in ((0, 5003), (1, 4001), (3, 5000), (8, 1000)):
        check(base[:, lo:hi], t, u, top_p=torch.full((9,), 0.9))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_logits(cuda, dtype):
    """Flat rows and rows of a few values: ties at every threshold go to the lowest indices."""
    V = 4000
    R = 24
    g = torch.Generator().manual_seed(3)
    flat = torch.full((R, V), 1.5).to(dtype)
    few = torch.randint(0, 4, (R, V), generator=g).to(dtype)
    u = torch.rand(R, generator=g, dtype=torch.float64)
    t = torch.ones(R)
    for x in (flat, few):
        check(x, t, u)
        check(x, t, u, top_k=torch.arange(1, R + 1).int() * 37)
        check(x, t, u, top_k=torch.full((R,), 700).int(), top_p=torch.arange(R) / R)
    # thresholds that fall on a whole number of equal weights
    check(flat, t, u, top_p=torch.full((R,), 0.5))
    got = run(flat, t, torch.full((R,), 0.9999), top_p=torch.full((R,), 0.25))
    assert (got == 999).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_nan_and_masks(cuda, dtype):
    g = torch.Generator().manual_seed(4)
    V = 3000
    x = (torch.randn(12, V, generator=g) * 2).to(dtype)
    low = torch.finfo(dtype).min
    x[0] = float("-inf")                                   # nothing left: every token alike
    x[1] = float("-inf")
    x[1, 2222] = -3.0                                      # one token left
    x[2, 7] = x[2, 1999] = float("inf")                    # the infinite ones share everything
    x[3, ::2] = float("nan")                               # no numbers: never drawn
    x[4] = low                                             # the type's lowest value everywhere
    x[5] = low
    x[5, 100:105] = 1.0
    x[6, 50:] = float("-inf")
    x[7] = float("nan")
    x[8] = torch.finfo(dtype).max
    x[9, :] = -0.0
    x[9, ::3] = 0.0
    u = torch.rand(12, generator=g)
    t = torch.tensor([1.0, 0.5, 1.0, 1.0, 1.0, 1.0, 0.7, 1.0, 1.0, 1.0, 1e-30, 3e38])
    none = dict(top_k=None, top_p=None, min_p=None)
    check(x, t, u, **none)
    check(x, t, u, top_k=torch.full((12,), 5).int())
    check(x, t, u, top_p=torch.full((12,), 0.5), min_p=torch.full((12,), 0.01))
    got = run(x, torch.zeros(12), u)                       # greedy: torch's argmax, NaN above everything
    assert got.tolist() == [sampling.argmax(r) for r in x.float().numpy()]
    assert got.tolist() == x.float().argmax(-1).tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [1, 2, 31, 33, 127, 129, 256, 257, 513, 1000, 1900, 2047, 2049, 5000])
@pytest.mark.parametrize("V", [700, 2500, 40001])
def test_short_lists(cuda, V, k, dtype):
    """Around the sizes at which a top-k goes from one list to the next, with equal logits that overflow them."""
    R = 8
    x, g = rows(R, V, dtype, V + k)
    x[1] = x[1].round()                                    # some tens of values
    x[2] = (x[2] > 2).to(dtype)                            # two values
    x[3] = 1.5
    x[4, V // 2:] = float("-inf")
    x[5, : V - 20] = x[5, : V - 20].sort(descending=True)[0]   # every large one in one place
    x[6, ::7] = 30.0
    u = torch.rand(R, generator=g)
    t = torch.rand(R, generator=g) + 0.3
    top_k = torch.full((R,), k).int()
    check(x, t, u, top_k=top_k)
    check(x, t, u, top_k=top_k, top_p=torch.rand(R, generator=g), min_p=torch.rand(R, generator=g) * 1e-3)
    check(x, t, u, top_p=torch.rand(R, generator=g), min_p=torch.rand(R, generator=g) * 1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_rows_than_start_at_once(cuda, dtype):
    """Rows begin in the order of their work there, each with its own settings."""
    R, V = 700, 5001
    x, g = rows(R, V, dtype, 12)
    pick = lambda xs: torch.tensor(xs)[torch.randint(len(xs), (R,), generator=g)]  # noqa: E731
    check(x, pick([0.0, 0.7, 1.0]), torch.rand(R, generator=g), top_k=pick([0, 0, 20, 400]).int(),
          top_p=pick([0.5, 0.9, 1.0]), min_p=pick([0.0, 0.0, 0.05]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1e-3, 1e-6, 1e-9, 1e-20, 1e-38, 1.0])
@pytest.mark.parametrize("scale", [1.0, 1e4, 1e10, 1e37])
def test_steps_of_the_type_against_the_temperature(cuda, dtype, t, scale):
    """Logits whose neighbours in the type lie many temperatures apart: the largest alone has a weight."""
    V = 9001
    x, g = rows(6, V, dtype, 8)
    x = (x.double() * scale).to(dtype)
    x[1, ::3] = float("-inf")
    x[2, 5:] = float("-inf")
    x[3] = x[3, 0]
    x[3, 17] = float("-inf")
    x[4] = -x[4].abs()
    x[4, 4000:] = float("-inf")
    x[5, 1::2] = torch.finfo(dtype).min
    u = torch.rand(6, generator=g)
    temp = torch.full((6,), t)
    check(x, temp, u)
    check(x, temp, u, top_k=torch.full((6,), 50).int(), top_p=torch.full((6,), 0.9))
    check(x, temp, u, min_p=torch.full((6,), 1e-30))


def test_extreme_settings(cuda):
    x, g = rows(10, 5000, torch.float32, 6)
    one = torch.ones(10)
    best = x.argmax(-1)
    u = torch.rand(10, generator=g)
    assert torch.equal(run(x, one, u, top_k=torch.ones(10).int()), best)
    assert torch.equal(run(x, one, u, top_p=torch.zeros(10)), best)
    assert torch.equal(run(x, one, u, min_p=one), best)
    assert torch.equal(run(x, one, u, min_p=one * 7), best)
    assert torch.equal(run(x, one * -1, u), best) and torch.equal(run(x, one * float("nan"), u), best)
    off = dict(top_k=torch.full((10,), -1).int(), top_p=one * 2, min_p=-one)
    assert torch.equal(run(x, one, u, **off), run(x, one, u))
    assert torch.equal(run(x, one, u, top_k=torch.full((10,), 5000).int()), run(x, one, u))
    # the ends of the uniform numbers' range, and numbers outside it
    kept = dict(top_k=torch.full((10,), 3).int())
    three = x.topk(3).indices.sort(-1).values
    assert torch.equal(run(x, one, torch.zeros(10), **kept), three[:, 0])
    assert torch.equal(run(x, one, one * 1.5, **kept), three[:, 2])
    assert torch.equal(run(x, one, one * float("nan"), **kept), three[:, 0])
    assert torch.equal(run(x, one, -one, **kept), three[:, 0])
    check(x, one * float("inf"), u)                         # an infinite temperature: all alike


def test_low_temperatures_and_far_ranks(cuda):
    """top-k whose last rank lies far below the maximum, and weights that vanish."""
    x, g = rows(8, 30000, torch.float32, 7)
    u = torch.rand(8, generator=g)
    check(x, torch.full((8,), 0.05), u, top_k=torch.full((8,), 20000).int())
    check(x, torch.full((8,), 0.01), u, top_p=torch.full((8,), 0.999))
    check(x * 1000, torch.full((8,), 1.0), u, top_k=torch.full((8,), 25000).int(), top_p=torch.full((8,), 0.9999))


# ---------------------------------------------------------------------------------------------- drafts
def run_verify(x, d, nd, t, au, u, dtype=torch.int64, **kw):
    from nvattn import ops
    dev = {k: v.cuda() for k, v in kw.items()}
    a, n = ops.verify_sampled(x.cuda(), d.to(dtype).cuda(), nd.to(dtype).cuda(), t.cuda(), au.cuda(), u.cuda(), **dev)
    assert a.dtype == n.dtype == dtype
    return a.cpu(), n.cpu()


def check_verify(x, d, nd, t, au, u, dtype=torch.int64, **kw):
    a, n = run_verify(x, d, nd, t, au, u, dtype, **kw)
    S, K = d.shape
    host = x.float().numpy().reshape(S, K + 1, -1)
    for s in range(S):
        want = sampling.verify(host[s], d[s].tolist(), int(nd[s]), float(t[s]), au[s].double().tolist(), float(u[s]),
                               *(kw[k][s].item() if k in kw else z for k, z in (("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))))
        assert (int(a[s]), int(n[s])) == want, s
    return a, n


@pytest.mark.parametrize("S,K,V,dtype", [(1, 1, 50, torch.float32), (7, 2, 1000, torch.bfloat16),
                                         (33, 4, 5001, torch.float32), (3, 8, 151936, torch.bfloat16),
                                         (5, 0, 300, torch.bfloat16)])
def test_verify(cuda, S, K, V, dtype):
    x, g = rows(S * (K + 1), V, dtype, S * 17 + K)
    x[:, ::97] += 4
    likely = x.float().view(S, K + 1, V)[:, :K].argmax(-1)
    d = torch.where(torch.rand(S, K, generator=g) < 0.7, likely, torch.randint(0, V, (S, K), generator=g))
    nd = torch.randint(0, K + 1, (S,), generator=g)
    nd[::2] = K
    t = torch.rand(S, generator=g) + 0.3
    t[2::4] = 0
    au, u = torch.rand(S, K, generator=g) * 0.7, torch.rand(S, generator=g)
    check_verify(x, d, nd, t, au, u)
    check_verify(x, d, nd, t, au.double(), u.double(), torch.int32, top_k=torch.randint(1, 40, (S,), generator=g).int(),
                 top_p=torch.rand(S, generator=g) * 0.5 + 0.5)
    check_verify(x, d, nd, t, au, u, min_p=torch.full((S,), 0.05))


def test_verify_drafts_at_the_edges(cuda):
    """Drafts outside the vocabulary, drafts that the settings removed, a draft that holds all the weight, the same
    token drafted again, ties with the draft among them."""
    V = 600
    x, g = rows(6 * 3, V, torch.float32, 9)
    d = x.view(6, 3, V)[:, :2].argmax(-1)
    d[0, 0] = V
    d[1, 0] = -1
    d[2, 0] = x.view(6, 3, V)[2, 0].argmin()                # removed by top-k
    d[3] = d[3, 0]
    x[4 * 3:] = 0.25                                       # flat rows: ties at the cut, the draft among them
    d[4, 0], d[5, 0] = 9, 10
    nd, one = torch.full((6,), 2), torch.ones(6)
    au, u = torch.full((6, 2), 0.05), torch.rand(6, generator=g)
    k = torch.full((6,), 10).int()
    check_verify(x, d, nd, one, au, u, top_k=k)
    check_verify(x, d, nd, one, au, u, top_k=torch.ones(6).int())
    check_verify(x, d, nd, one, torch.full((6, 2), 0.9999), u, top_k=k, top_p=torch.full((6,), 0.7))


def test_greedy_verify_is_verify_drafts_greedy(cuda):
    from nvattn.sampler import verify_drafts_greedy, verify_drafts_sampled
    x, g = rows(20 * 4, 3001, torch.bfloat16, 10)
    x = (x * 2).round().cuda()                              # many ties
    d = x.view(20, 4, -1)[:, :3].argmax(-1)
    d[::3, 1] += 1
    nd = torch.randint(0, 4, (20,), generator=g).cuda()
    z = torch.zeros(20, device="cuda")
    want = verify_drafts_greedy(x, d, nd)
    got = verify_drafts_sampled(x, d, nd, z, torch.zeros(20, 3, device="cuda"), z)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_speculation_draws_like_sampling(cuda):
    """Over a grid of both uniform numbers: a token comes out (accepted or drawn instead) with its own probability."""
    V, N = 9, 256
    logits = torch.randn(1, V, generator=torch.Generator().manual_seed(11)) * 1.5
    w = sampling.kept_weights(logits[0].numpy(), 0.8, top_p=0.95)
    p = torch.from_numpy(w / w.sum())
    grid = (torch.arange(N) + 0.5) / N
    x = logits.repeat(2 * N * N, 1)
    d = torch.full((N * N, 1), 4)
    one = torch.ones(N * N)
    a, n = run_verify(x, d, one.long(), one * 0.8, grid.repeat_interleave(N)[:, None], grid.repeat(N),
                      top_p=one * 0.95)
    first = torch.where(a > 0, d[:, 0], n)
    freq = torch.bincount(first, minlength=V).double() / (N * N)
    assert float((freq - p).abs().max()) <= 2 / N           # a grid of N points is off by 1 / N per boundary


def test_replayed_graph_and_another_stream(cuda):
    from nvattn import ops, sampler
    S, K, V = 16, 3, 20000
    x, g = rows(S * (K + 1), V, torch.bfloat16, 12)
    xd = x.cuda()
    u, au = torch.zeros(S, device="cuda"), torch.zeros(S, K, device="cuda")
    t = torch.full((S,), 0.9, device="cuda")
    p = torch.full((S,), 0.9, device="cuda")
    d = xd.float().view(S, K + 1, V)[:, :K].argmax(-1)
    nd = torch.full((S,), K, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ids = sampler.sample_tokens(xd[:S], t, u, top_p=p)
            held = ops.verify_sampled(xd, d, nd, t, au, u, top_p=p)
        for _ in range(4):
            u.copy_(torch.rand(S, generator=g))
            au.copy_(torch.rand(S, K, generator=g))
            graph.replay()
            want = sampler.sample_tokens(xd[:S], t, u, top_p=p), *ops.verify_sampled(xd, d, nd, t, au, u, top_p=p)
            for a, b in zip((ids, *held), want):
                assert torch.equal(a, b)
    side.synchronize()
    check(x[:S], t.cpu(), u.cpu(), top_p=p.cpu(), got=ids.cpu())


def test_no_rows(cuda):
    from nvattn import ops, sampler
    e = torch.zeros(0, device="cuda")
    assert sampler.sample_tokens(torch.zeros(0, 50, device="cuda"), e, e).shape == (0,)
    a, n = ops.verify_sampled(torch.zeros(0, 50, device="cuda"), torch.zeros(0, 2, dtype=torch.int64, device="cuda"),
                              torch.zeros(0, dtype=torch.int64, device="cuda"), e, torch.zeros(0, 2, device="cuda"), e)
    assert a.shape == n.shape == (0,)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_plain_verify_at_segment_edges(cuda, dtype):
    """Drafts in the first and last tokens of a warp's segment, as the only token, without a weight and out of range."""
    V, S, K = 9000, 12, 2
    x, g = rows(S * (K + 1), V, dtype, 41)
    d = torch.tensor([[0, V - 1], [1023, 1024], [2047, 2048], [4095, 4096], [8191, 8192], [V - 1, 0], [5, 5], [-1, V],
                      [77, 78], [1024, 2048], [8999, 8998], [3, 2047]])
    row = x.view(S, K + 1, V)
    for s in range(8):                                     # often accepted: most of the weight
        for j in range(K):
            if 0 <= d[s, j] < V:
                row[s, j, d[s, j]] = 16.0
    row[8] = float("-inf")                                 # nothing but the draft
    row[8, 0, 77] = row[8, 1, 78] = row[8, 2, 4] = 0.5
    row[9, :, 1024] = float("-inf")                        # drafts without a weight
    row[10, 0] = float("-inf")                             # nothing at all: every token alike
    row[11, 0, :2048] = float("-inf")                      # the draft alone in its segment
    row[11, 0, 3] = 6.0
    nd = torch.full((S,), K)
    one = torch.ones(S)
    for hi in (0.5, 0.999, 1.0):
        au, u = torch.rand(S, K, generator=g) * hi, torch.rand(S, generator=g)
        check_verify(x, d, nd, one, au, u)
        check_verify(x, d, nd, one * 0.6, au.double(), u.double(), torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_plain_rows_of_any_alignment(cuda, dtype):
    """Rows that begin at any element, with a stride of their own: the same draws as packed ones."""
    R, V = 9, 5003
    x, g = rows(R, V, dtype, 43)
    u, t = torch.rand(R, generator=g), torch.rand(R, generator=g) + 0.3
    t[4] = 0
    want = check(x, t, u)
    for first, stride in ((1, V + 1), (3, V + 6), (8, V + 5)):
        big = torch.full((first + R * stride,), 50.0, dtype=dtype, device="cuda")
        view = big[first:].as_strided((R, V), (stride, 1))
        view.copy_(x)
        assert torch.equal(run(view, t, u), want)


def test_calls_on_two_streams_at_once(cuda):
    from nvattn.sampler import sample_tokens
    x, g = rows(40, 30011, torch.float32, 44)
    x, u, t = x.cuda(), torch.rand(40, generator=g).cuda(), torch.rand(40, generator=g).cuda() + 0.3
    p = torch.full((40,), 0.8, device="cuda")
    k = torch.full((40,), 60, dtype=torch.int32, device="cuda")
    settings = [dict(), dict(top_p=p), dict(top_k=k), dict(top_k=k, top_p=p)]
    want = [sample_tokens(x, t, u, **s) for s in settings]
    streams = [torch.cuda.Stream() for _ in settings]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, kw in zip(streams, settings):
            with torch.cuda.stream(s):
                got.append(sample_tokens(x, t, u, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_of_two_host_threads(cuda):
    """Calls of very different sizes from threads at once: the shared memory that one asks for does not limit the
    other's.  Through the C ABI, so that the threads are in the library at the same time for the most part."""
    import threading
    from nvattn import _lib
    from nvattn.sampler import sample_tokens
    lib = _lib.load()
    cases = []
    for R, V in ((1, 151936), (70, 1000), (1, 151936), (70, 1000)):
        x, g = rows(R, V, torch.float32, V)
        x, t, p, u = (a.cuda() for a in (x, torch.ones(R), torch.full((R,), 0.9), torch.rand(R, generator=g)))
        cases.append((x, t, u, p, sample_tokens(x, t, u, top_p=p), torch.cuda.Stream()))
    torch.cuda.synchronize()
    failed = []

    def work(x, t, u, p, want, stream):
        ids = torch.empty_like(want)
        args = (x.data_ptr(), x.shape[1], x.shape[0], x.shape[1], 4, t.data_ptr(), 0, p.data_ptr(), 0, u.data_ptr(), 4,
                ids.data_ptr(), 0, 0, stream.cuda_stream)
        torch.cuda.set_device(0)
        status = [lib.nva_sample_tokens(*args) for _ in range(8000)]
        stream.synchronize()
        if any(status) or not torch.equal(ids, want):
            failed.append((x.shape, sum(s != 0 for s in status)))

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert failed == []


@pytest.mark.parametrize("V,dtype", [(393216, torch.float32), (393216, torch.bfloat16), (262144, torch.float32)])
def test_the_largest_vocabularies(cuda, V, dtype):
    """Up to the largest that the calls take (include/nvattn.h), whose rows fill the shared memory of eight CTAs."""
    R = 2
    x, g = rows(R, V, dtype, 77)
    u, t = torch.rand(R, generator=g, dtype=torch.float64), torch.rand(R, generator=g) + 0.4
    check(x, t, u)
    check(x, t, u, top_p=torch.full((R,), 0.95))
    check(x, t, u, top_k=torch.tensor([50, 6000]).int(), min_p=torch.full((R,), 0.001))
    d = torch.stack([x[0].argmax(), x[1].argmin()]).view(2, 1)
    check_verify(x.repeat_interleave(2, 0), d, torch.ones(2, dtype=torch.int64), t, torch.full((2, 1), 0.001), u.float(),
                 top_p=torch.full((R,), 0.95))
