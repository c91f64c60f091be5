"""Paged key-value cache: append, attention of one new token and eviction against plain 64-bit forms (serving_ref.py,
which derives the bounds)."""
import math

import numpy as np
import pytest
import torch

import serving_ref as R
from grxcp_b200 import _native as N
from grxcp_b200 import dnn as D

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def attend(dnn, lens, kv_heads, group, dim, page, dtype, heads_first=False, window=0, weights=False, room=None, seed=0, q_scale=1.0,
           lse=True):
    room = max(lens + [1]) if room is None else room
    k, v, table, tokens = R.make_cache(lens, room, kv_heads, dim, page, dtype, heads_first, seed)
    cache = D.PagedCache(k, v, table)
    g = torch.Generator().manual_seed(seed + 1)
    q = (q_scale * torch.randn(len(lens), kv_heads * group, dim, generator=g)).to(dtype)
    o = torch.full((len(lens), kv_heads * group, 1, dim), math.nan, dtype=dtype, device="cuda")
    got_lse = torch.full((len(lens), kv_heads * group), math.nan, device="cuda") if lse else None
    w0 = torch.rand(len(lens), kv_heads, cache.capacity + 5, generator=g)
    w = w0.cuda() if weights else None
    scale = dim ** -0.5
    torch.cuda.synchronize()  # the handle may be on another stream than the inputs
    assert dnn.paged_attention(cache, ints(lens), q.cuda()[:, :, None], o, scale, window, got_lse, w) == N.SUCCESS
    torch.cuda.synchronize()
    assert dnn.execution_status() == N.SUCCESS
    for b, r in enumerate(R.attention(tokens, q, scale, window, dtype)):
        err = (o[b, :, 0].cpu().double() - r["o"]).abs()
        assert (err <= r["o_tol"]).all(), (b, (err - r["o_tol"]).max().item())
        if lse:
            x = got_lse[b].cpu().double()
            if lens[b] == 0:
                assert (x == -math.inf).all()
            else:
                assert ((x - r["lse"]).abs() <= r["lse_tol"]).all()
        if weights:
            x, want = w[b].cpu().double(), w0[b].double()
            seen = slice(r["first"], lens[b])
            assert ((x[:, seen] - want[:, seen] - r["w"]).abs() <= r["w_tol"] + 2.0 ** -23).all()
            x[:, seen] = want[:, seen]
            assert torch.equal(x, want), "a slot that no query sees has changed"
    return o, got_lse, w


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 2, 4), (64, 3, 1), (256, 1, 16), (128, 1, 8), (64, 2, 7), (128, 2, 1), (256, 2, 2)])
def test_attention_heads(dnn, dtype, dim, kv_heads, group):
    attend(dnn, [1, 0, 17, 130, 333, 64], kv_heads, group, dim, 16, dtype, weights=True)


@pytest.mark.parametrize("group", [17, 24, 32, 40])
def test_attention_many_heads_on_one(dnn, group):
    attend(dnn, [5, 200, 31], 1, group, 128, 16, BF, weights=True)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 48, 64, 128, 300])
@pytest.mark.parametrize("heads_first", [False, True])
def test_attention_pages(dnn, page, heads_first):
    attend(dnn, [15, 16, 33, 1, 257], 2, 4, 128, page, BF, heads_first, weights=True)


@pytest.mark.parametrize("window", [1, 5, 16, 63, 100, 5000])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_window(dnn, window, dim):
    attend(dnn, [0, 1, 100, 163, 700], 2, 4, dim, 20, BF, True, window, weights=True)


@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 0], [2049], [4000, 1, 0, 9], list(range(0, 260, 2)), [700] * 40])
def test_attention_lengths(dnn, lens):
    attend(dnn, lens, 2, 4, 128, 16, BF, room=max(lens) + 40, weights=True)
    attend(dnn, lens, 1, 1, 64, 32, HF, lse=False)


def test_attention_long_and_peaked(dnn):
    """Few rows, a long cache, and scores that spread over dozens of units, so that joined parts differ much."""
    attend(dnn, [40_003, 12_345], 1, 8, 128, 64, BF, weights=True, q_scale=8.0)
    attend(dnn, [30_001], 2, 2, 64, 16, HF, True, q_scale=6.0)


def test_attention_many_sequences(dnn):
    lens = [(i * 37) % 91 for i in range(700)]
    attend(dnn, lens, 1, 2, 64, 16, BF, weights=True)


def test_attention_repeats_bit_for_bit(dnn):
    lens = [3000, 17, 900, 0, 1500]
    a = attend(dnn, lens, 2, 4, 128, 16, BF, weights=True)
    b = attend(dnn, lens, 2, 4, 128, 16, BF, weights=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_attention_strided_and_row_of_minus_infinity(dnn):
    """q and o inside wider buffers; scores of -inf for some keys, which then weigh nothing."""
    k, v, table, _ = R.make_cache([40], 48, 1, 128, 16, BF)
    row = table[0].long()
    k[row[0], 3, 0] = 0
    k[row[0], 3, 0, 0] = -math.inf
    buf = torch.randn(1, 7, 4, 256, device="cuda").to(BF)
    q = buf[:, 2:3, :, 64:192].transpose(1, 2)
    q[..., 0] = 1.0
    out = torch.full((1, 7, 4, 256), 3.0, device="cuda", dtype=BF)
    o = out[:, 5:6, :, 128:].transpose(1, 2)
    lse = torch.empty(1, 4, device="cuda")
    assert dnn.paged_attention(D.PagedCache(k, v, table), ints([40]), q, o, 0.1, 0, lse) == N.SUCCESS
    kk, vv = (x[row].flatten(0, 1)[:40, 0].double() for x in (k, v))
    p = torch.softmax(q[0, :, 0].double() @ kk.T * 0.1, 1)
    assert p[:, 3].max() == 0
    assert torch.allclose(o[0, :, 0].double(), p @ vv, atol=2e-2, rtol=2e-2)
    out[:, 5:6, :, 128:] = 3.0
    assert (out == 3.0).all()
    assert torch.isfinite(lse).all()


def test_attention_bad_page_is_reported_and_skipped(dnn):
    k, v, table, tokens = R.make_cache([40, 20], 48, 2, 64, 16, BF)
    want = table.clone()
    table[0, 1] = 10 ** 6
    q = torch.randn(2, 4, 1, 64, device="cuda").to(BF)
    o = torch.empty_like(q)
    assert dnn.paged_attention(D.PagedCache(k, v, table), ints([40, 20]), q, o, 0.125) == N.SUCCESS
    assert dnn.execution_status() == N.EXECUTION_FAILED
    assert dnn.execution_status() == N.SUCCESS
    kept = [torch.cat([x[:16], x[32:]]) for x in tokens[0]]
    for b, r in enumerate(R.attention([kept, tokens[1]], q[:, :, 0].cpu(), 0.125, 0, BF)):
        assert ((o[b, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
    assert dnn.paged_attention(D.PagedCache(k, v, want), ints([40, 20]), q, o, 0.125) == N.SUCCESS
    assert dnn.execution_status() == N.SUCCESS


def test_lengths_out_of_range_are_clamped(dnn):
    k, v, table, tokens = R.make_cache([48, 20], 48, 1, 64, 16, BF)
    q = torch.randn(2, 2, 1, 64, device="cuda").to(BF)
    o, lse = torch.empty_like(q), torch.empty(2, 2, device="cuda")
    assert dnn.paged_attention(D.PagedCache(k, v, table), ints([2 ** 31 - 1, -5]), q, o, 0.125, 0, lse) == N.SUCCESS
    r = R.attention(tokens, q[:, :, 0].cpu(), 0.125, 0, BF)[0]
    assert ((o[0, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
    assert (o[1] == 0).all() and (lse[1] == -math.inf).all()


def test_offsets_past_32_bits(dnn):
    """Pages more than 2^31 elements into their pools."""
    page, dim = 64, 128
    pages = 2 ** 31 // (page * dim) + 8
    k, v = (torch.zeros(pages, page, 1, dim, dtype=BF, device="cuda") for _ in range(2))
    table = ints([[pages - 1, 2, pages - 3]])
    kb, vb = (torch.randn(1, 1, 150, dim, device="cuda").to(BF) for _ in range(2))
    cache, lens = D.PagedCache(k, v, table), ints([0])
    assert dnn.kv_append(cache, lens, kb, vb, None, lens) == N.SUCCESS
    assert torch.equal(k[pages - 1, :, 0], kb[0, 0, :64]) and torch.equal(v[pages - 3, :22, 0], vb[0, 0, 128:])
    q = torch.randn(1, 4, 1, dim, device="cuda").to(BF)
    o = torch.empty_like(q)
    assert dnn.paged_attention(cache, lens, q, o, 0.1) == N.SUCCESS
    r = R.attention([(kb[0].transpose(0, 1).cpu(), vb[0].transpose(0, 1).cpu())], q[:, :, 0].cpu(), 0.1, 0, BF)[0]
    assert ((o[0, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
    w = torch.rand(1, 1, cache.capacity, device="cuda")
    kept = R.evict(w[0, 0].cpu().numpy(), 150, 70, 10)
    assert dnn.kv_evict(cache, lens, w, 70, 10) == N.SUCCESS
    assert torch.equal(torch.cat([k[pages - 1, :, 0], k[2, :6, 0]]), kb[0, 0][kept])
    assert lens.item() == 70 and dnn.execution_status() == N.SUCCESS


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("tokens,page,heads,dim,heads_first", [(1, 16, 8, 128, False), (1, 1, 3, 64, True), (5, 3, 2, 256, True),
                                                               (300, 64, 2, 128, False), (1000, 20, 1, 64, True), (17, 16, 16, 256, False)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(dnn, tokens, page, heads, dim, heads_first, ragged):
    lens = [0, 1, 15, 16, 77]
    k, v, table, _ = R.make_cache(lens, 80 + tokens, heads, dim, page, BF, heads_first, poison=False)
    want_k, want_v = k.clone(), v.clone()
    counts = [min(tokens, c) for c in (0, 1, tokens // 2, tokens, max(0, tokens - 1))] if ragged else [tokens] * 5
    new_k = torch.randn(5, tokens, heads, dim, device="cuda").to(BF).transpose(1, 2)
    new_v = torch.randn(5, heads, tokens, dim, device="cuda").to(BF)
    for b in range(5):
        for t in range(counts[b]):
            at = lens[b] + t
            p = table[b, at // page]
            want_k[p, at % page] = new_k[b, :, t]
            want_v[p, at % page] = new_v[b, :, t]
    held, out = ints(lens), ints([-7] * 5)
    cache = D.PagedCache(k, v, table)
    assert dnn.kv_append(cache, held, new_k, new_v, ints(counts) if ragged else None, out) == N.SUCCESS
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert out.tolist() == [n + c for n, c in zip(lens, counts)] and held.tolist() == lens
    assert dnn.kv_append(cache, held, new_k, new_v, ints(counts) if ragged else None, held) == N.SUCCESS  # over its own lengths
    assert held.tolist() == out.tolist()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert dnn.execution_status() == N.SUCCESS


def test_append_past_the_room(dnn):
    k, v, table, _ = R.make_cache([40, 10], 48, 2, 64, 16, BF, poison=False)
    before = k.clone()
    new = torch.randn(2, 2, 20, 64, device="cuda").to(BF)
    lens = ints([40, 10])
    assert dnn.kv_append(D.PagedCache(k, v, table), lens, new, new, None, lens) == N.SUCCESS
    assert dnn.execution_status() == N.EXECUTION_FAILED
    assert lens.tolist() == [48, 30]
    p = table[0, 2].long()
    assert torch.equal(k[p, 8:], new[0, :, :8].transpose(0, 1)) and torch.equal(k[p, :8], before[p, :8])


# ---------------------------------------------------------------- eviction

def run_evict(dnn, lens, keep, recent, heads=2, dim=64, page=16, in_place=False, heads_first=False, weights=None, page_out=None, dtype=BF,
              indices=True):
    room = max(max(lens), keep, 1)
    k, v, table, tokens = R.make_cache(lens, room, heads, dim, page, dtype, heads_first, poison=False)
    cache = D.PagedCache(k, v, table)
    g = torch.Generator().manual_seed(5)
    w = torch.exp(2 * torch.randn(len(lens), heads, cache.capacity + 3, generator=g)) if weights is None else weights(cache.capacity)
    w_dev, held = w.cuda(), ints(lens)
    idx = torch.full((len(lens), heads, keep), -9, dtype=torch.int32, device="cuda") if indices else None
    if in_place:
        out, lens_out, w_out, ko, vo = cache, held, w_dev, k, v
        assert dnn.kv_evict(cache, held, w_dev, keep, recent, indices=idx) == N.SUCCESS
    else:
        ko, vo, to, _ = R.make_cache([0] * len(lens), keep, heads, dim, page_out or page, dtype, heads_first, 9, poison=False)
        out = D.PagedCache(ko, vo, to)
        lens_out, w_out = ints([-3] * len(lens)), torch.full((len(lens), heads, out.capacity + 7), 5.0, device="cuda")
        src = k.clone(), v.clone(), w_dev.clone()
        assert dnn.kv_evict(cache, held, w_dev, keep, recent, out, lens_out, w_out, idx) == N.SUCCESS
        assert torch.equal(k, src[0]) and torch.equal(v, src[1]) and torch.equal(w_dev.nan_to_num(7.0), src[2].nan_to_num(7.0))
    assert lens_out.tolist() == [min(n, keep) for n in lens]
    size, rows = out.desc.pageSize, out.page_table.cpu()
    ko, vo, w_out = ko.cpu(), vo.cpu(), w_out.cpu()
    for b, n in enumerate(lens):
        m = min(n, keep)
        at = torch.arange(m)
        pages = rows[b].long()[at // size] if m else at
        for h in range(heads):
            kept = R.evict(w[b, h].numpy(), n, keep, recent)
            if indices:
                assert idx[b, h].tolist() == kept + [-1] * (keep - m), (b, h)
            assert torch.equal(ko[pages, at % size, h], tokens[b][0][kept, h])
            assert torch.equal(vo[pages, at % size, h], tokens[b][1][kept, h])
            assert torch.equal(w_out[b, h, :m].nan_to_num(7.0), w[b, h][kept].nan_to_num(7.0))
            assert (w_out[b, h, m:out.capacity] == 0).all()
            tail = w_out[b, h, out.capacity:]
            assert torch.equal(tail.nan_to_num(7.0), w[b, h, out.capacity:].nan_to_num(7.0)) if in_place else (tail == 5.0).all()
    assert dnn.execution_status() == N.SUCCESS


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (64, 0), (64, 64), (100, 17), (333, 50), (1000, 1000)])
def test_evict_budgets(dnn, keep, recent, in_place):
    run_evict(dnn, [0, 1, 63, 64, 65, 333, 700], keep, recent, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("heads,dim,page,heads_first", [(1, 128, 1, False), (3, 256, 20, True), (8, 128, 64, True), (2, 64, 300, False)])
def test_evict_layouts(dnn, heads, dim, page, heads_first, in_place):
    run_evict(dnn, [500, 40, 301], 200, 31, heads, dim, page, in_place, heads_first)


def test_evict_into_other_pages_and_without_indices(dnn):
    run_evict(dnn, [500, 40], 200, 31, page=16, page_out=24, dtype=HF)
    run_evict(dnn, [500, 40], 200, 31, page=24, page_out=16, indices=False)
    run_evict(dnn, [500, 40], 200, 31, in_place=True, indices=False)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,keep", [(5000, 4999), (20_011, 1777), (70_001, 30_000)])
def test_evict_long(dnn, n, keep, in_place):
    run_evict(dnn, [n], keep, 64, heads=1, page=64, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["zero", "few", "special", "close", "rising", "falling"])
def test_evict_ties_and_special_weights(dnn, kind, in_place):
    def weights(cap):
        g = torch.Generator().manual_seed(3)
        w = torch.rand(3, 2, cap + 1, generator=g)
        i = torch.arange(cap + 1).float()
        if kind == "zero":
            return torch.zeros_like(w)
        if kind == "few":
            return (w * 4).floor()
        if kind == "close":
            return 1.0 + (w * 9).floor() * 2.0 ** -23
        if kind in ("rising", "falling"):
            return (i if kind == "rising" else -i).expand(3, 2, -1).contiguous()
        pick = torch.randint(0, 6, w.shape, generator=g)
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5])
        return torch.where(torch.rand(w.shape, generator=g) < 0.7, special[pick], w - 0.5)
    run_evict(dnn, [2500, 130, 129], 128, 9, in_place=in_place, weights=weights)


# ------------------------------------------------- streams, graphs, scratch

def test_two_streams_of_one_handle(dnn):
    """The handle moves between streams without a wait: each stream's scratch is its own."""
    lens = [6000, 2500]
    k, v, table, tokens = R.make_cache(lens, 6000, 1, 128, 16, BF)
    cache, held = D.PagedCache(k, v, table), ints(lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.randn(2, 8, 1, 128, device="cuda").to(BF) for _ in range(2)]
    outs = [torch.empty_like(q) for q in qs]
    ws = [torch.zeros(2, 1, cache.capacity, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, o, w in zip(streams, qs, outs, ws):
            dnn.set_stream(s)
            assert dnn.paged_attention(cache, held, q, o, 0.09, 0, None, w) == N.SUCCESS
    torch.cuda.synchronize()
    dnn.set_stream(None)
    for q, o, w in zip(qs, outs, ws):
        for b, r in enumerate(R.attention(tokens, q[:, :, 0].cpu(), 0.09, 0, BF)):
            assert ((o[b, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
            assert ((w[b, :, :lens[b]].cpu().double() / 20 - r["w"]).abs() <= 2 * r["w_tol"]).all()


def test_decoding_loop_in_a_graph(dnn):
    """append, attention and eviction captured once and replayed: lengths live on the device, and the scratch that the
    capture made outlives a later call that needs more."""
    room, keep = 96, 64
    k, v, table, _ = R.make_cache([0, 0], room, 2, 64, 16, BF, poison=False)
    cache, lens = D.PagedCache(k, v, table), ints([90, 3])
    w = torch.zeros(2, 2, cache.capacity, device="cuda")
    nk, nv = (torch.randn(2, 2, 1, 64, device="cuda").to(BF) for _ in range(2))
    q = torch.randn(2, 4, 1, 64, device="cuda").to(BF)
    o = torch.empty_like(q)
    assert dnn.kv_append(cache, ints([0, 0]), nk, nv) == N.SUCCESS  # binds the handle to its device

    def step():
        D.check(dnn.kv_append(cache, lens, nk, nv, None, lens))
        D.check(dnn.paged_attention(cache, lens, q, o, 0.125, 0, None, w))
        D.check(dnn.kv_evict(cache, lens, w, keep, 8))

    start = [x.clone() for x in (k, v, lens, w)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    dnn.set_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    attend(dnn, [5000], 1, 8, 128, 16, BF, weights=True)
    with torch.cuda.stream(s):
        for x, y in zip((k, v, lens, w), start):
            x.copy_(y)
        for _ in range(70):
            graph.replay()
        got = [x.clone() for x in (k, v, lens, w, o)]
        for x, y in zip((k, v, lens, w), start):
            x.copy_(y)
        for _ in range(70):
            step()
    torch.cuda.synchronize()
    dnn.set_stream(None)
    assert lens.tolist() == [keep, keep]
    assert all(torch.equal(x, y) for x, y in zip(got, (k, v, lens, w, o)))
    assert dnn.execution_status() == N.SUCCESS


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,keep,recent", [(40_000, 20_001, 3), (17_001, 16_900, 0), (70_001, 5, 2)])
def test_evict_few_long_sequences(dnn, n, keep, recent, in_place):
    """Few heads of long sequences: several CTAs share a selection, and a move."""
    def weights(cap):
        g = torch.Generator().manual_seed(8)
        return (torch.rand(2, 2, cap + 1, generator=g) * 1000).floor()  # ties everywhere, across the CTAs' runs
    run_evict(dnn, [n, n // 3], keep, recent, heads=2, page=64, in_place=in_place, weights=weights)


def test_attention_hands_on_nan_and_infinity_of_its_own(dnn):
    """What a query sees is not hidden: a NaN in q or in a seen key gives NaN, as the formula does; other heads and
    sequences stay what they are."""
    lens = [300, 50, 1000]
    k, v, table, tokens = R.make_cache(lens, 1000, 1, 128, 16, BF)
    q = torch.randn(3, 4, 1, 128, device="cuda").to(BF)
    clean, o = torch.empty_like(q), torch.empty_like(q)
    cache = D.PagedCache(k, v, table)
    w = torch.zeros(3, 1, cache.capacity, device="cuda")
    assert dnn.paged_attention(cache, ints(lens), q, clean, 0.09) == N.SUCCESS
    q[1, 2, 0, 5] = math.nan
    k[table[2, 40].long(), 3] = math.nan  # token 643 of the last sequence
    lse = torch.zeros(3, 4, device="cuda")
    assert dnn.paged_attention(cache, ints(lens), q, o, 0.09, 0, lse, w) == N.SUCCESS
    nan = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    nan[1, 2] = nan[2] = True
    assert torch.equal(torch.isnan(lse), nan) and torch.equal(torch.isnan(o[:, :, 0]).all(2), nan)
    assert torch.equal(o[~nan], clean[~nan])
    assert torch.isfinite(w[0]).all() and torch.isnan(w[1, 0, :50]).all()


def test_cache_views(dnn):
    """K and V interleaved in one tensor, heads that are some of a wider pool's, a page table inside a wider one."""
    lens, dim = [70, 33], 64
    k, v, table, tokens = R.make_cache(lens, 80, 2, dim, 16, HF, poison=False)
    both = torch.full((k.shape[0], 16, 2, 6, dim), math.nan, device="cuda", dtype=HF)
    both[:, :, 0, 3:5], both[:, :, 1, 3:5] = k, v
    wide = torch.full((2, table.shape[1] + 9), 10 ** 8, device="cuda", dtype=torch.int32)
    wide[:, 4:4 + table.shape[1]] = table
    cache = D.PagedCache(both[:, :, 0, 3:5], both[:, :, 1, 3:5], wide[:, 4:4 + table.shape[1]])
    q = torch.randn(2, 6, 1, dim, device="cuda").to(HF)
    o = torch.empty_like(q)
    assert dnn.paged_attention(cache, ints(lens), q, o, 0.125) == N.SUCCESS
    for b, r in enumerate(R.attention(tokens, q[:, :, 0].cpu(), 0.125, 0, HF)):
        assert ((o[b, :, 0].cpu().double() - r["o"]).abs() <= r["o_tol"]).all()
    held, w = ints(lens), torch.rand(2, 2, cache.capacity, device="cuda")
    kept = R.evict(w[0, 1].cpu().numpy(), 70, 40, 5)
    assert dnn.kv_evict(cache, held, w, 40, 5) == N.SUCCESS
    rows = table[0].long()
    assert torch.equal(both[rows, :, 1, 4].flatten(0, 1)[:40].cpu(), tokens[0][1][kept, 1])
    new = torch.randn(2, 2, 3, dim, device="cuda").to(HF)
    assert dnn.kv_append(cache, held, new, new, None, held) == N.SUCCESS
    assert torch.equal(both[rows, :, 0, 3].flatten(0, 1)[40:43], new[0, 0]) and held.tolist() == [43, 36]
    assert torch.isnan(both[:, :, :, :3]).all() and torch.isnan(both[:, :, :, 5]).all()
    assert dnn.execution_status() == N.SUCCESS


def test_a_failed_allocation_is_reported_and_passes(monkeypatch, dev):
    with D.Handle() as h:
        k, v, table, _ = R.make_cache([20], 32, 1, 64, 16, BF)
        cache, lens = D.PagedCache(k, v, table), ints([20])
        q = torch.randn(1, 1, 1, 64, device="cuda").to(BF)
        w = torch.rand(1, 1, cache.capacity, device="cuda")
        assert h.kv_append(cache, ints([0]), k[:1, :1].transpose(1, 2), v[:1, :1].transpose(1, 2), ints([0])) == N.SUCCESS
        monkeypatch.setenv("GRX_FAULT_INJECT", "alloc")
        assert h.paged_attention(cache, lens, q, q, 0.125) == N.ALLOC_FAILED
        assert h.kv_evict(cache, lens, w, 10, 2) == N.ALLOC_FAILED
        monkeypatch.delenv("GRX_FAULT_INJECT")
        assert h.paged_attention(cache, lens, q, q, 0.125) == N.SUCCESS
        assert h.kv_evict(cache, lens, w, 10, 2) == N.SUCCESS and lens.item() == 10


def test_ragged_batches_share_by_share(dnn):
    """Lengths whose tiles are cut in many ways between CTAs: within items, at their ends, and right behind."""
    g = torch.Generator().manual_seed(2)
    for trial in range(6):
        lens = torch.randint(0, 3000 if trial % 2 else 300, (40 + 50 * trial,), generator=g).tolist()
        lens[3] = 9000
        attend(dnn, lens, 2, 4, 64, 32, BF, weights=trial % 3 == 0, seed=trial)
