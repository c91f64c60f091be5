"""Whose scratch a serving call uses: graphs that are replayed beside one another, threads' default streams, streams that
come and go. Every result is checked against the plain forms of serving_ref.py."""
import ctypes
import math
import threading
import time

import pytest
import torch

import serving_ref as R
from grxcp_b200 import _native as N
from grxcp_b200 import dnn as D

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
LENS, SCALE = [6000, 2500], 0.09  # cut between many CTAs, whose parts are joined


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Work:
    """Attention over a shared cache, its weights added up, and an eviction into a cache of its own."""

    def __init__(self, cache, tokens, held, seed):
        g = torch.Generator().manual_seed(seed)
        self.cache, self.tokens, self.held, self.calls = cache, tokens, held, 0
        self.q = torch.randn(2, 8, 1, 128, generator=g).to(BF).cuda()
        self.o = torch.full_like(self.q, math.nan)
        self.lse = torch.full((2, 8), math.nan, device="cuda")
        self.w = torch.zeros(2, 1, cache.capacity, device="cuda")
        self.fixed = torch.rand(2, 1, cache.capacity, generator=g).cuda()
        k, v, table, _ = R.make_cache([0, 0], 700, 1, 128, 16, BF, seed=seed, poison=False)
        self.out, self.out_lens = D.PagedCache(k, v, table), ints([0, 0])
        self.out_w = torch.zeros(2, 1, self.out.capacity, device="cuda")

    def run(self, dnn, evict=True):
        D.check(dnn.paged_attention(self.cache, self.held, self.q, self.o, SCALE, 0, self.lse, self.w))
        if evict:
            D.check(dnn.kv_evict(self.cache, self.held, self.fixed, 700, 50, self.out, self.out_lens, self.out_w))

    def check(self, calls, evict=True):
        for b, r in enumerate(R.attention(self.tokens, self.q[:, :, 0].cpu(), SCALE, 0, BF)):
            assert ((self.o[b, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
            assert ((self.lse[b].cpu().double() - r["lse"]).abs() <= r["lse_tol"]).all()
            # each addition to a weight is rounded once: calls * 2^-24 of at most itself more
            assert ((self.w[b, :, :LENS[b]].cpu().double() / calls - r["w"]).abs() <= r["w_tol"] + calls * 2.0 ** -24 * r["w"]).all()
            if evict:
                kept = R.evict(self.fixed[b, 0].cpu().numpy(), LENS[b], 700, 50)
                at = torch.arange(700)
                rows = self.out.page_table[b].cpu().long()[at // 16]
                assert torch.equal(self.out.k_pages.cpu()[rows, at % 16, 0], self.tokens[b][0][kept, 0])
                assert torch.equal(self.out_w[b, 0, :700].cpu(), self.fixed[b, 0].cpu()[kept])


@pytest.fixture()
def shared(dev):
    k, v, table, tokens = R.make_cache(LENS, 6000, 1, 128, 16, BF)
    return D.PagedCache(k, v, table), tokens, ints(LENS)


def test_graphs_of_one_stream_beside_one_another(dnn, shared):
    """Two graphs captured on one stream, replayed on two others, and plain calls on the first meanwhile."""
    works = [Work(*shared, seed) for seed in (1, 2, 3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    dnn.set_stream(streams[2])
    works[2].run(dnn)
    torch.cuda.synchronize()
    graphs = []
    for w in works[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=streams[2]):
            for _ in range(3):
                w.run(dnn)
    torch.cuda.synchronize()
    for _ in range(25):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for _ in range(3):
            works[2].run(dnn)
    torch.cuda.synchronize()
    dnn.set_stream(None)
    for w, calls in zip(works, (75, 75, 76)):
        w.check(calls)
    assert dnn.execution_status() == N.SUCCESS


def test_threads_on_their_default_streams(dnn, shared):
    """One stream handle (cudaStreamPerThread), a stream for each thread."""
    works = [Work(*shared, seed) for seed in (4, 5, 6)]
    torch.cuda.synchronize()
    dnn.set_stream(2)
    failed = []

    def loop(w):
        try:
            for _ in range(40):
                w.run(dnn)
        except Exception as e:
            failed.append(e)
    threads = [threading.Thread(target=loop, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    dnn.set_stream(None)
    assert not failed
    for w in works:
        w.check(40)


def test_streams_that_come_and_go(dnn, shared):
    """A stream is destroyed while its work is under way; the next one may get its handle."""
    cuda = ctypes.CDLL("libcuda.so.1")
    works = [Work(*shared, seed) for seed in (7, 8)]
    torch.cuda.synchronize()
    for i in range(12):
        s = ctypes.c_void_p()
        assert cuda.cuStreamCreate(ctypes.byref(s), 1) == 0
        dnn.set_stream(s.value)
        for _ in range(5):
            works[i % 2].run(dnn, evict=False)
        dnn.set_stream(None)
        if i % 2:  # an even and an odd one's work lie beside each other, works of one kind do not
            torch.cuda.synchronize()
        assert cuda.cuStreamDestroy_v2(s) == 0
    torch.cuda.synchronize()
    for w in works:
        w.check(30, evict=False)


def test_a_graph_gives_its_scratch_back(dnn):
    """64 MiB of scores a capture (16 query heads, room for 2^20 tokens), for one graph after the other."""
    page = 64
    k, v = (torch.randn(2, page, 1, 64, device="cuda").to(BF) for _ in range(2))
    table = torch.full((1, (1 << 20) // page), -1, dtype=torch.int32, device="cuda")
    table[0, :2] = ints([1, 0])
    cache, held = D.PagedCache(k, v, table), ints([100])
    q = torch.randn(1, 16, 1, 64, device="cuda").to(BF)
    o, lse, w = torch.empty_like(q), torch.empty(1, 16, device="cuda"), torch.zeros(1, 1, 1 << 20, device="cuda")
    keys = torch.cat([k[1, :, 0], k[0, :36, 0]]).double()
    want = torch.logsumexp(q[0, :, 0].double() @ keys.T * 0.125, 1)
    assert dnn.paged_attention(cache, held, q, o, 0.125, 0, lse, w) == N.SUCCESS
    s = torch.cuda.Stream()
    dnn.set_stream(s)
    free = []
    for _ in range(14):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            D.check(dnn.paged_attention(cache, held, q, o, 0.125, 0, lse, w))
        lse.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(lse[0].double(), want, atol=1e-3)
        graph.reset()
        time.sleep(0.1)  # a thread of CUDA's tells the graph's end, when it comes to it
        free.append(torch.cuda.mem_get_info()[0])
    dnn.set_stream(None)
    assert free[1] - free[-1] < 3 * (64 << 20), free


def test_a_call_in_a_capture_that_has_failed(dnn, shared):
    """It says so, and the stream's calls after it are what they were."""
    cuda = ctypes.CDLL("libcuda.so.1")
    w = Work(*shared, 9)
    s, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert cuda.cuStreamCreate(ctypes.byref(s), 1) == 0
    torch.cuda.synchronize()
    dnn.set_stream(s.value)
    w.run(dnn)
    assert cuda.cuStreamBeginCapture_v2(s, 2) == 0  # relaxed
    assert cuda.cuStreamSynchronize(s) != 0  # not allowed in a capture, which has failed now
    assert dnn.paged_attention(w.cache, w.held, w.q, w.o, SCALE) == N.EXECUTION_FAILED
    assert cuda.cuStreamEndCapture(s, ctypes.byref(graph)) != 0
    for _ in range(3):
        w.run(dnn)
    torch.cuda.synchronize()
    dnn.set_stream(None)
    assert cuda.cuStreamDestroy_v2(s) == 0
    w.check(4)
