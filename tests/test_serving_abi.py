"""CPU checks of the serving entry points: bad arguments are refused before any device is touched, empty problems are
SUCCESS, and the Python mirror refuses tensors that the raw calls would misread."""
import ctypes as C

import pytest
import torch

from grxcp_b200 import _native as N
from grxcp_b200 import dnn as D

P = 1 << 20  # any aligned non-null address: validation returns before it is touched
L = N.lib


@pytest.fixture()
def h():
    with D.Handle() as hh:
        yield hh.h


def cache(**kw):
    c = N.grxdnnPagedCache_t(2, 4, 128, 10, 16, 5, 5, 16 * 4 * 128, 4 * 128, 128, N.GRX_R_16BF)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rows(heads=4, seq=1, dim=128, batch=2, dtype=N.GRX_R_16BF, **kw):
    d = D.attn_desc(None, batch, heads, seq, dim, dtype)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_CACHE = [(dict(batch=-1), 3), (dict(kvHeads=0), 3), (dict(headDim=0), 3), (dict(numPages=0), 3), (dict(pageSize=0), 3),
             (dict(maxPages=0), 3), (dict(strideTable=4), 3), (dict(pageSize=1 << 20, maxPages=1 << 12, strideTable=1 << 12), 3),
             (dict(stridePage=64), 3), (dict(strideToken=64), 3), (dict(strideHead=-128), 3), (dict(dtype=N.GRX_R_32F), 6),
             (dict(dtype=N.GRX_R_8F_E4M3), 6), (dict(strideToken=516), 6), (dict(strideHead=129), 6), (dict(stridePage=8193), 6)]


@pytest.mark.parametrize("change,status", BAD_CACHE)
def test_cache_descriptor(h, change, status):
    c, good = cache(**change), cache()
    q, kv = rows(8, batch=c.batch), rows(c.kvHeads, dim=c.headDim, batch=c.batch)
    q.headDim = kv.headDim = c.headDim
    q.dtype = kv.dtype = c.dtype
    r = C.byref
    assert L.grxdnnPagedAttentionForward(h, r(c), P, P, P, P, r(q), P, r(q), P, 0.1, 0, None, None, 0) == status
    assert L.grxdnnKvCacheAppend(h, r(c), P, P, P, P, r(kv), P, r(kv), P, None, None) == status
    same = [getattr(c, f) == getattr(good, f) for f in ("batch", "kvHeads", "headDim")]
    for a, b in ((c, good), (good, c)) if all(same) else ((c, c),):
        assert L.grxdnnKvCacheEvict(h, r(a), P, P, P, P, P, 1 << 33, 32, 4, r(b), P, P, P, P, P, 1 << 33, None) == status


def test_head_dim(h):
    for dim in (32, 96, 192, 512):
        c = cache(headDim=dim, strideHead=dim, strideToken=4 * dim, stridePage=64 * dim)
        q = rows(8, dim=dim)
        assert L.grxdnnPagedAttentionForward(h, C.byref(c), P, P, P, P, C.byref(q), P, C.byref(q), P, 0.1, 0, None, None, 0) == 6


def test_attention(h):
    c, q = cache(), rows(8)

    def call(hh=h, c=c, k=P, v=P, table=P, lens=P, qd=q, q=P, od=q, o=P, scale=0.1, window=0, weights=None, pitch=0):
        ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return L.grxdnnPagedAttentionForward(hh, ref(c), k, v, table, lens, ref(qd), q, ref(od), o, scale, window, None, weights, pitch)
    assert call(hh=None) == N.NOT_INITIALIZED
    for k in ("c", "qd", "od", "k", "v", "table", "lens", "q", "o"):
        assert call(**{k: None}) == N.INVALID_VALUE, k
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == N.INVALID_VALUE
    assert call(window=-1) == N.INVALID_VALUE
    assert call(weights=P, pitch=79) == N.INVALID_VALUE  # room for 80 tokens
    assert call(qd=rows(6), od=rows(6)) == N.INVALID_VALUE  # 6 query heads on 4
    for other in (rows(4), rows(8, batch=3), rows(8, dim=64), rows(8, seq=2)):
        assert call(od=other) == N.INVALID_VALUE
    assert call(qd=rows(8, seq=2), od=rows(8, seq=2)) == N.NOT_SUPPORTED
    assert call(qd=rows(8, dtype=N.GRX_R_16F)) == N.NOT_SUPPORTED
    assert call(od=rows(8, dtype=N.GRX_R_32F)) == N.NOT_SUPPORTED
    assert call(q=P + 8) == N.NOT_SUPPORTED and call(o=P + 2) == N.NOT_SUPPORTED and call(k=P + 4) == N.NOT_SUPPORTED
    assert call(qd=rows(8, strideHead=130)) == N.NOT_SUPPORTED
    assert call(qd=rows(0), od=rows(0)) == N.SUCCESS
    assert call(c=cache(batch=0), qd=rows(8, batch=0), od=rows(8, batch=0)) == N.SUCCESS


def test_append(h):
    c, kv = cache(), rows(4, seq=3)

    def call(hh=h, c=c, kp=P, vp=P, table=P, lens=P, kd=kv, k=P, vd=kv, v=P, counts=None, out=None):
        ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return L.grxdnnKvCacheAppend(hh, ref(c), kp, vp, table, lens, ref(kd), k, ref(vd), v, counts, out)
    assert call(hh=None) == N.NOT_INITIALIZED
    for k in ("c", "kd", "vd", "kp", "vp", "table", "lens", "k", "v"):
        assert call(**{k: None}) == N.INVALID_VALUE, k
    for other in (rows(8, seq=3), rows(4, seq=2), rows(4, seq=3, dim=64), rows(4, seq=3, batch=1), rows(4, seq=3, strideSeq=64)):
        assert call(vd=other) == N.INVALID_VALUE
    assert call(kd=rows(4, seq=3, dtype=N.GRX_R_16F)) == N.NOT_SUPPORTED
    assert call(k=P + 2) == N.NOT_SUPPORTED and call(vd=rows(4, seq=3, strideSeq=132)) == N.NOT_SUPPORTED
    empty = rows(4, seq=0)
    assert call(kd=empty, k=None, vd=empty, v=None) == N.SUCCESS
    none = rows(4, seq=3, batch=0)
    assert call(c=cache(batch=0), kd=none, vd=none) == N.SUCCESS


def test_evict(h):
    def call(hh=h, c=cache(), k=P, table=P, lens=P, w=P, pitch=80, keep=32, recent=4, o=cache(), ko=P, to=P, lo=P, wo=P, po=80):
        ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return L.grxdnnKvCacheEvict(hh, ref(c), k, P, table, lens, w, pitch, keep, recent, ref(o), ko, P, to, lo, wo, po, None)
    assert call(hh=None) == N.NOT_INITIALIZED
    for k in ("c", "k", "table", "lens", "w", "o", "ko", "to", "lo", "wo"):
        assert call(**{k: None}) == N.INVALID_VALUE, k
    assert call(pitch=79) == N.INVALID_VALUE and call(po=79) == N.INVALID_VALUE
    assert call(keep=0) == N.INVALID_VALUE and call(recent=33) == N.INVALID_VALUE and call(recent=-1) == N.INVALID_VALUE
    assert call(keep=81, recent=0) == N.INVALID_VALUE  # more than the output cache has room for
    assert call(o=cache(batch=1)) == N.INVALID_VALUE and call(o=cache(kvHeads=2)) == N.INVALID_VALUE
    assert call(o=cache(dtype=N.GRX_R_16F)) == N.NOT_SUPPORTED
    assert call(ko=P + 8) == N.NOT_SUPPORTED
    assert call(c=cache(batch=0), o=cache(batch=0)) == N.SUCCESS


def test_scores(h):
    def call(hh=h, r=4, v=1000, x=P, t=N.GRX_R_16BF, ld=1000, scale=1.0, tok=P, logp=P, ent=None, lse=None, k=0, tt=None, tl=None):
        return L.grxdnnTokenLogProbsForward(hh, r, v, x, t, ld, scale, tok, logp, ent, lse, k, tt, tl)
    assert call(hh=None) == N.NOT_INITIALIZED
    for kw in (dict(r=-1), dict(v=-1), dict(v=0), dict(x=None), dict(ld=999), dict(scale=0.0), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(tok=None), dict(k=-1), dict(k=33, tt=P), dict(v=8, k=9, tt=P)):
        assert call(**kw) == N.INVALID_VALUE, kw
    assert call(t=N.GRX_R_8I) == N.NOT_SUPPORTED
    assert call(r=0, x=None) == N.SUCCESS
    assert call(logp=None, tok=None) == N.SUCCESS  # nothing asked for


def test_score_gradient(h):
    def call(hh=h, r=4, v=1000, x=P, t=N.GRX_R_16BF, ld=1000, scale=1.0, tok=P, lse=P, ent=None, dl=P, de=None, dx=2 * P,
             dt=N.GRX_R_16BF, ldd=1000):
        return L.grxdnnTokenLogProbsBackward(hh, r, v, x, t, ld, scale, tok, lse, ent, dl, de, dx, dt, ldd)
    assert call(hh=None) == N.NOT_INITIALIZED
    for kw in (dict(r=-1), dict(v=0), dict(x=None), dict(dx=None), dict(lse=None), dict(ld=999), dict(ldd=999), dict(scale=-1.0),
               dict(dl=None), dict(tok=None), dict(de=P), dict(dx=P, ldd=1001)):
        assert call(**kw) == N.INVALID_VALUE, kw
    assert call(t=N.GRX_R_8I, dt=N.GRX_R_8I) == N.NOT_SUPPORTED and call(dt=N.GRX_R_32F) == N.NOT_SUPPORTED
    assert call(r=0, x=None) == N.SUCCESS


def test_python_mirror_refuses_what_it_would_misread():
    k = torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        D.PagedCache(k, k.float(), table)
    with pytest.raises(ValueError):
        D.PagedCache(k, k.transpose(1, 2).contiguous().transpose(1, 2), table)
    with pytest.raises(ValueError):
        D.PagedCache(k, k, table.long())
    with pytest.raises(ValueError):
        D.PagedCache(k, k, table.T)
    c = D.PagedCache(k, k, table)
    q = torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16)
    lens, w = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 32)
    with D.Handle() as h:
        for bad in (lens.long(), lens[:2], torch.zeros(6, dtype=torch.int32)[::2]):
            with pytest.raises(ValueError):
                h.paged_attention(c, bad, q, q, 0.1)
            with pytest.raises(ValueError):
                h.kv_append(c, lens, q[:, :2], q[:, :2], counts=bad)
        with pytest.raises(ValueError):
            h.paged_attention(c, lens, q, q, 0.1, lse=torch.zeros(3, 3))
        for bad in (w.double(), w[:, :1], w[..., ::2], w[0]):
            with pytest.raises(ValueError):
                h.paged_attention(c, lens, q, q, 0.1, weights=bad)
            with pytest.raises(ValueError):
                h.kv_evict(c, lens, bad, 4, 1)
        with pytest.raises(ValueError):
            h.kv_evict(c, lens, w, 4, 1, out=c)
        with pytest.raises(ValueError):
            h.kv_evict(c, lens, w, 4, 1, indices=torch.zeros(3, 2, 5, dtype=torch.int32))
        x, t, f = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
        for bad in (dict(tokens=t.long()), dict(logp=f.double()), dict(logp=f[:3]), dict(logits=x.T), dict(top_tokens=t),
                    dict(top_tokens=torch.zeros(4, 2, dtype=torch.int32), top_logp=torch.zeros(4, 3))):
            with pytest.raises(ValueError):
                h.token_logprobs(**{**dict(logits=x, tokens=t, logp=f), **bad})
        with pytest.raises(ValueError):
            h.token_logprobs_backward(x, t, f, f, x[:, :9])
