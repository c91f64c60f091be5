"""Paged cache on a GPU: buffers that are their own output, lengths and pages written right before they are read, captures
with a fresh handle."""
import math

import pytest
import torch

import serving_ref as R
from grxcp_b200 import _native as N
from grxcp_b200 import dnn as D

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n,keep", [(40_000, 20_001), (9_000, 4_000), (1_000, 900)])
def test_evict_into_other_pages_with_weights_over_themselves(dnn, n, keep):
    """The pools are others', lengths and weights their own output: the CTAs that share a head still read a weight before
    one of them writes over it."""
    lens = [n, n // 2 + 7]
    k, v, table, tokens = R.make_cache(lens, n, 1, 64, 64, BF, poison=False)
    ko, vo, to, _ = R.make_cache([0, 0], keep, 1, 64, 64, BF, seed=3, poison=False)
    cache, out = D.PagedCache(k, v, table), D.PagedCache(ko, vo, to)
    slots = max(cache.capacity, out.capacity) + 1
    g = torch.Generator().manual_seed(4)
    for _ in range(10):
        w = torch.rand(2, 1, slots, generator=g)
        w_dev, held = w.cuda(), ints(lens)
        assert dnn.kv_evict(cache, held, w_dev, keep, 30, out, held, w_dev) == N.SUCCESS
        got = w_dev.cpu()
        for b, m in enumerate(lens):
            kept = R.evict(w[b, 0].numpy(), m, keep, 30)
            assert torch.equal(got[b, 0, :len(kept)], w[b, 0][kept])
            assert (got[b, 0, len(kept):out.capacity] == 0).all() and torch.equal(got[b, 0, out.capacity:], w[b, 0, out.capacity:])
            at = torch.arange(len(kept))
            assert torch.equal(ko.cpu()[to[b].cpu().long()[at // 64], at % 64, 0], tokens[b][0][kept, 0])
        assert held.tolist() == [min(m, keep) for m in lens]
    assert dnn.execution_status() == N.SUCCESS


def test_lengths_in_pinned_memory(dnn):
    """Pinned host memory has one address for both sides and stays open to the calls; the same tensor unpinned is refused."""
    k, v, table, tokens = R.make_cache([40, 7], 48, 1, 64, 16, BF)
    q = torch.randn(2, 2, 1, 64, device="cuda").to(BF)
    o = torch.empty_like(q)
    lens = torch.tensor([40, 7], dtype=torch.int32)
    with pytest.raises(ValueError, match="^lens must be on the GPU"):
        dnn.paged_attention(D.PagedCache(k, v, table), lens, q, o, 0.125)
    assert dnn.paged_attention(D.PagedCache(k, v, table), lens.pin_memory(), q, o, 0.125) == N.SUCCESS
    torch.cuda.synchronize()
    for b, r in enumerate(R.attention(tokens, q[:, :, 0].cpu(), 0.125, 0, BF)):
        assert ((o[b, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()


def test_capture_with_a_fresh_handle(dev):
    """The first call of a handle, which binds it to its device and allocates, may be a captured one."""
    k, v, table, tokens = R.make_cache([70, 30], 96, 1, 64, 16, BF, poison=False)
    cache, lens = D.PagedCache(k, v, table), ints([70, 30])
    q = torch.randn(2, 4, 1, 64, device="cuda").to(BF)
    o, w = torch.empty_like(q), torch.zeros(2, 1, cache.capacity, device="cuda")
    x, t = torch.randn(5, 3001, device="cuda"), ints([1, 2, 3, 4, 5])
    logp = torch.empty(5, device="cuda")
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with D.Handle() as h:
        h.set_stream(s)
        with torch.cuda.graph(graph, stream=s):
            status = [h.paged_attention(cache, lens, q, o, 0.125, weights=w), h.kv_evict(cache, lens, w, 60, 10),
                      h.token_logprobs(x, t, logp)]
        assert status == [N.SUCCESS] * 3
        graph.replay()
        torch.cuda.synchronize()
        for b, r in enumerate(R.attention(tokens, q[:, :, 0].cpu(), 0.125, 0, BF)):
            assert ((o[b, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
        assert lens.tolist() == [60, 30]
        assert torch.allclose(logp, torch.log_softmax(x, 1).gather(1, t.long()[:, None])[:, 0], atol=1e-4)
        assert h.execution_status() == N.SUCCESS
        del graph


@pytest.mark.parametrize("batch,weights", [(1, False), (3, True), (64, False)])
def test_lengths_and_pages_written_right_before(dnn, batch, weights):
    """Lengths that an append or an eviction writes, and a table that changes, right before the attention that reads them.
    With keys of 0 every score is 0 and lse tells the length; the values tell the pages."""
    page, room, steps = 16, 400, 300
    g = torch.Generator().manual_seed(6)
    pages = batch * (room // page)
    k = torch.zeros(2 * pages, page, 1, 64, device="cuda", dtype=BF)
    v = torch.cat([torch.full((pages, page, 1, 64), c, device="cuda", dtype=BF) for c in (1.0, 2.0)])
    tables = [(torch.randperm(pages, generator=g) + c * pages).to(torch.int32).reshape(batch, -1).cuda() for c in (0, 1)]
    table = tables[0].clone()
    cache = D.PagedCache(k, v, table)
    lens = ints([(37 * b) % 300 for b in range(batch)])
    w = torch.zeros(batch, 1, cache.capacity, device="cuda")
    q = torch.randn(batch, 2, 1, 64, device="cuda").to(BF)
    lse = torch.empty(steps, batch, 2, device="cuda")
    o = torch.empty(steps, batch, 2, 1, 64, device="cuda", dtype=BF)
    new = [torch.zeros(batch, 1, 1, 64, device="cuda", dtype=BF), torch.ones(batch, 1, 1, 64, device="cuda", dtype=BF)]
    n, want = lens.tolist(), []
    for i in range(steps):
        D.check(dnn.kv_append(cache, lens, new[0], new[i % 2] + 1 if i % 2 else new[1], None, lens))
        D.check(dnn.paged_attention(cache, lens, q, o[i], 0.125, 0, lse[i], w if weights else None))
        n = [x + 1 for x in n]
        want.append(list(n))
        if i % 7 == 6:
            D.check(dnn.kv_evict(cache, lens, w, 200, 150))
            n = [min(x, 200) for x in n]
        table.copy_(tables[(i + 1) % 2])  # the next step's pages: all values 1, then all 2
    torch.cuda.synchronize()
    assert dnn.execution_status() == N.SUCCESS
    assert torch.allclose(lse, torch.log(torch.tensor(want, device="cuda").float())[..., None].expand_as(lse), atol=1e-4)
    assert lens.tolist() == n
    assert (o[0::2] == 1).all() and (o[1::2] == 2).all()
