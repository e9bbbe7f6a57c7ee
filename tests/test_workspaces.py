"""Which workspace an attention call takes (nvattn.ops._workspace): calls that may overlap never share one.  The host
side without a GPU, and calls in flight together on one."""
import contextlib

import pytest
import torch


# ---------------------------------------------------------------------------------------------- the choice (no GPU)
class _Sizes:
    """The library's size queries, without a device."""
    nva_varlen_workspace_bytes = staticmethod(lambda *a: 100)
    nva_paged_decode_workspace_bytes = staticmethod(lambda *a: 200)
    nva_paged_attention_fp8_workspace_bytes = staticmethod(lambda *a: 300)


@pytest.fixture()
def at(monkeypatch):
    """Sets the current stream's number and whether it is capturing."""
    from nvattn import _lib, ops
    now = {"stream": 0, "capturing": False}
    monkeypatch.setattr(ops, "_raw_stream", lambda index: now["stream"], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    monkeypatch.setattr(ops, "_on", lambda device: ops._HERE)
    monkeypatch.setattr(_lib, "load", lambda: _Sizes)
    monkeypatch.setattr(ops, "_WORKSPACES", {})
    monkeypatch.setattr(ops, "_RETIRED", [])

    def go(stream, capturing=False):
        now.update(stream=stream, capturing=capturing)
    return go


DEV = torch.device("cpu", 0)    # (a device with an index; nothing here runs on it)


def test_each_stream_has_its_own(at):
    from nvattn import ops
    at(0)
    default = ops._workspace(64, DEV)
    at(7)
    one = ops._workspace(64, DEV)
    at(9)
    other = ops._workspace(64, DEV)
    assert len({x.data_ptr() for x in (default, one, other)}) == 3
    assert all(int(x.count_nonzero()) == 0 for x in (default, one, other))
    at(7)
    assert ops._workspace(32, DEV) is one
    at(0)
    assert ops._workspace(64, DEV) is default


def test_captured_calls_share_none_with_eager_ones(at):
    from nvattn import ops
    at(0)
    default = ops._workspace(64, DEV)
    at(7)
    one = ops._workspace(64, DEV)
    at(7, capturing=True)
    graph = ops._workspace(64, DEV)
    assert graph is not default and graph is not one
    at(9, capturing=True)
    assert ops._workspace(64, DEV) is graph
    with pytest.raises(RuntimeError, match="reserve_workspace"):
        ops._workspace(65, DEV)


def test_own_workspace(at, monkeypatch):
    """Whatever the stream's number: torch gives the same ones out again."""
    import threading
    from nvattn import ops
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    at(0)
    assert ops.reserve_workspace(4, 64, 32, 8, device=DEV) == 200
    assert ops.reserve_workspace(4, 64, 32, 8, device=DEV, fp8_cache=True) == 300
    mine = torch.zeros(ops.workspace_bytes(4, 64, 32, 8, fp8_cache=True), dtype=torch.uint8).view(-1)
    dev = mine.device
    other = []
    at(9, capturing=True)
    shared = ops._workspace(300, DEV)
    with ops.own_workspace(mine):
        assert ops._workspace(300, dev) is mine
        with pytest.raises(RuntimeError, match="301 bytes"):
            ops._workspace(301, dev)
        with pytest.raises(RuntimeError, match="cpu:0"):
            ops._workspace(300, DEV)                                   # (another device)
        thread = threading.Thread(target=lambda: other.append(ops._workspace(300, DEV)))
        thread.start()
        thread.join()
    assert other[0] is shared and ops._workspace(300, DEV) is shared


def test_growing_keeps_what_graphs_hold(at):
    from nvattn import ops
    at(0)
    ops._workspace(64, DEV)
    at(7, capturing=True)
    small = ops._workspace(64, DEV)
    at(0)
    ops._workspace(128, DEV)
    at(7, capturing=True)
    assert ops._workspace(128, DEV) is not small and any(x is small for x in ops._RETIRED)


@pytest.mark.parametrize("fp8", [True, False])
def test_host_threads_take_turns(at, monkeypatch, fp8):
    """The kernels of a call follow one another through one workspace: no other thread's call begins between them."""
    import threading
    import time
    from nvattn import _lib, ops
    inside, worst = [0], [0]

    class Lib(_Sizes):
        def __getattr__(self, name):
            def call(*args):
                inside[0] += 1
                worst[0] = max(worst[0], inside[0])
                time.sleep(0.01)
                inside[0] -= 1
                return 0
            return call

    monkeypatch.setattr(_lib, "load", lambda: Lib())
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    at(0)
    workspace = ops._workspace
    monkeypatch.setattr(ops, "_workspace", lambda nbytes, device: workspace(nbytes, DEV))
    c = torch.zeros(2, 256, 8, 128, dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16)
    kw = dict(zip(("k_scale", "v_scale"), ops.kvcache_scales(c))) if fp8 else {}
    q, lens = torch.zeros(3, 1, 32, 128, dtype=torch.bfloat16), torch.ones(3, dtype=torch.int32)
    cu, table = torch.arange(4, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)

    def work():
        for _ in range(3):
            ops.flash_attn_with_kvcache(q, c, c, cache_seqlens=lens, block_table=table, softmax_scale=0.1, **kw)
            ops.flash_attn_varlen_func(q[:, 0], c, c, 1, cu, 1, cu, 0.1, block_table=table, **kw)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert worst[0] == 1


# ------------------------------------------------------------------------------------------- calls in flight together
def calls(seed, fp8):
    """A decode batch and a mixed one whose sequences are cut over many CTAs; returns a function that runs both."""
    from nvattn import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = [9000 + 700 * seed, 31, 2500]
    pages = [(x + 255) // 256 for x in lens]
    NB = sum(pages)
    kv = torch.randn(2, NB, 256, 8, 128, generator=g, device="cuda")
    cache = [x.to(torch.float8_e4m3fn) if fp8 else x.bfloat16() for x in kv]
    scales = dict(zip(("k_scale", "v_scale"), torch.ones(2, NB, 8, 16, device="cuda"))) if fp8 else {}
    table = torch.full((3, max(pages)), -1, dtype=torch.int32)
    order = torch.randperm(NB, generator=torch.Generator().manual_seed(seed)).int()
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    table = table.cuda()
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qlens = [300, 1, 9]
    cu = lambda xs: torch.tensor([0] + xs).cumsum(0).int().cuda()  # noqa: E731
    cu_q, cu_k = cu(qlens), cu(lens)
    q1 = torch.randn(3, 2, 32, 128, generator=g, device="cuda").bfloat16()
    q2 = torch.randn(sum(qlens), 32, 128, generator=g, device="cuda").bfloat16()

    def run(outs=(None, None)):
        return (ops.flash_attn_with_kvcache(q1, cache[0], cache[1], cache_seqlens=lens_d, block_table=table,
                                            softmax_scale=0.09, out=outs[0], **scales),
                ops.flash_attn_varlen_func(q2, cache[0], cache[1], max(qlens), cu_q, max(lens), cu_k, 0.09,
                                           block_table=table, out=outs[1], **scales))
    return run


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [True, False])
def test_streams_at_once(cuda, fp8):
    """Two streams in each other's way, neither waiting for the other: the bits that each gives alone."""
    from nvattn import _lib
    runs = [calls(1, fp8), calls(2, fp8)]
    want = [[x.clone() for x in r()] for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(runs[i]())
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        for outs in many:
            assert all(torch.equal(x, y) for x, y in zip(w, outs))
    assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [True, False])
def test_replays_beside_eager_calls_and_beside_each_other(cuda, fp8):
    """A graph on one stream, eager calls on another, a second graph, captured in a workspace of its own, on a third;
    both captured on the same stream."""
    from nvattn import _lib, ops
    runs = [calls(s, fp8) for s in (1, 2, 3)]
    want = [[x.clone() for x in r()] for r in runs]
    streams = [torch.cuda.Stream() for _ in range(3)]
    ops.reserve_workspace(8, 512, 32, 8, fp8_cache=fp8)
    own = torch.zeros(ops.workspace_bytes(8, 512, 32, 8, fp8_cache=fp8), dtype=torch.uint8, device="cuda")
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, run, w, within in zip(graphs, runs, want, (contextlib.nullcontext(), ops.own_workspace(own))):
        outs.append([torch.empty_like(x) for x in w])
        torch.cuda.synchronize()
        with within, torch.cuda.graph(graph):
            run(outs[-1])
    torch.cuda.synchronize()
    for _ in range(10):
        for o in outs:
            for x in o:
                x.zero_()
        torch.cuda.synchronize()
        eager = []
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            with torch.cuda.stream(streams[2]):
                eager.append(runs[2]())
        torch.cuda.synchronize()
        for got, w in list(zip(outs, want)) + [(e, want[2]) for e in eager]:
            assert all(torch.equal(x, y) for x, y in zip(got, w))
    assert _lib.device_error() == 0
