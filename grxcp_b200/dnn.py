"""grxDNN from Python: norms (forward and backward), softmax, GELU, conv2d, pooling, attention (forward and backward),
and token serving (paged key-value cache, attention of one new token, eviction, scoring of given tokens).

Thin mirror of include/grx/grxdnn.h; every method returns the raw status code
of the C call. Tensors are torch CUDA tensors (or integer device addresses).
"""
from __future__ import annotations

import ctypes as C
import struct

from . import _native as N
from ._native import lib
from .blas import CODES, dtype_code, ptr, stream_ptr


class GrxdnnError(RuntimeError):
    def __init__(self, status: int, what: str = ""):
        self.status = status
        super().__init__(f"{what}: {N.STATUS.get(status, status)} ({lib.grxdnnGetStatusString(status).decode()})")


def check(status: int, what: str = "grxdnn") -> None:
    if status != N.SUCCESS:
        raise GrxdnnError(status, what)


def attn_desc(t, batch=None, heads=None, seq=None, head_dim=None, dtype=None) -> N.grxdnnAttnTensor_t:
    """Descriptor of a [batch, heads, seq, head_dim] tensor (strides in elements)."""
    if t is not None and hasattr(t, "stride"):
        b, h, s, hd = t.shape
        sb, sh, ss, sd = t.stride()
        if sd != 1:
            raise ValueError("head_dim must be contiguous")
        return N.grxdnnAttnTensor_t(b, h, s, hd, sb, sh, ss, dtype_code(t))
    return N.grxdnnAttnTensor_t(batch, heads, seq, head_dim, heads * seq * head_dim, seq * head_dim, head_dim,
                                dtype if dtype is not None else N.GRX_R_16BF)


_ATTN = struct.Struct("@4i3qi0q").pack  # a grxdnnAttnTensor_t's bytes
assert len(_ATTN(*range(8))) == C.sizeof(N.grxdnnAttnTensor_t)


def _seen(t, name: str) -> None:
    """Refuses a tensor whose memory a kernel cannot read: a host address would fault on the GPU. Pinned memory has one
    address for both sides."""
    if not t.is_cuda and not t.is_pinned():
        raise ValueError(f"{name} must be on the GPU or pinned, not in {t.device} memory")


def _attn(t, name: str) -> bytes:
    """attn_desc of a tensor as plain bytes, which a C call takes too and which cost a third of it: for the calls that
    are made once a token."""
    b, h, s, hd = t.shape
    sb, sh, ss, sd = t.stride()
    if sd != 1:
        raise ValueError("head_dim must be contiguous")
    if not t.is_cuda:
        _seen(t, name)
    return _ATTN(b, h, s, hd, sb, sh, ss, CODES[t.dtype])  # filled when the cache of the call was made


def conv_desc(x, w, pad=(0, 0), stride=(1, 1), dilation=(1, 1)):
    n, h, wd, c = x.shape
    k, r, s, _ = w.shape
    return N.grxdnnConvDesc_t(n, h, wd, c, k, r, s, pad[0], pad[1], stride[0], stride[1], dilation[0], dilation[1])


def conv_out_dims(d) -> tuple[int, int]:
    p, q = C.c_int(), C.c_int()
    st = lib.grxdnnConvOutputDims(C.byref(d), C.byref(p), C.byref(q))
    if st != 0:
        raise ValueError(f"bad conv geometry (status {st})")
    return p.value, q.value


def pool_desc(x, window, pad=(0, 0), stride=(1, 1), mode=0):
    n, h, wd, c = x.shape
    return N.grxdnnPoolDesc_t(n, h, wd, c, window[0], window[1], pad[0], pad[1], stride[0], stride[1], mode)


def _array(t, kind: int, numel: int, name: str):
    """Address of a contiguous array of `numel` values: the raw calls take these by address alone, and would misread a
    tensor of another type, size or order."""
    if t is None or type(t) is int:
        return t
    if CODES.get(t.dtype) != kind or t.numel() != numel or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {N.TYPE_NAMES[kind]} with {numel} elements, not {t.dtype} {tuple(t.shape)}")
    if not t.is_cuda:
        _seen(t, name)
    return t.data_ptr()


_I32, _F32 = N.GRX_R_32I, N.GRX_R_32F


def _rows(t, name: str) -> tuple[int, int, int]:
    """Rows, columns and row pitch of a matrix."""
    rows, cols = t.shape
    pitch, step = t.stride()
    if cols > 1 and step != 1:
        raise ValueError(f"{name} rows must be contiguous")
    if not t.is_cuda:
        _seen(t, name)
    return rows, cols, pitch if rows > 1 else cols


class PagedCache:
    """A paged key-value cache: pools k_pages and v_pages [pages, page_size, kv_heads, head_dim] of equal strides (any
    order of the first three dimensions; head_dim contiguous) and a page table, int32 [batch, max_pages] with
    contiguous rows. Keeps the tensors and their descriptor, so that a decoding loop builds it once."""

    def __init__(self, k_pages, v_pages, page_table):
        code = dtype_code(k_pages)
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError("k_pages and v_pages must be [pages, page_size, kv_heads, head_dim] alike")
        if k_pages.stride() != v_pages.stride() or (k_pages.stride(3) != 1 and k_pages.shape[3] != 1):
            raise ValueError("k_pages and v_pages must have equal strides, head_dim contiguous")
        if page_table.dim() != 2 or CODES.get(page_table.dtype) != _I32:
            raise ValueError("page_table must be int32 [batch, max_pages]")
        if page_table.stride(1) != 1 and page_table.shape[1] != 1:
            raise ValueError("page_table rows must be contiguous")
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table
        pages, page, heads, dim = k_pages.shape
        sp, st, sh, _ = k_pages.stride()
        batch, width = page_table.shape
        self.batch, self.kv_heads, self.capacity = batch, heads, width * page
        self.desc = N.grxdnnPagedCache_t(batch, heads, dim, pages, page, width,
                                         max(width, page_table.stride(0)) if batch < 2 else page_table.stride(0),
                                         sp, st, sh, code)
        self.ref = C.byref(self.desc)
        self.k, self.v, self.table = k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr()
        # Whether kernels can read it all; a cache that they cannot is refused by the calls that use it.
        self.seen = all(t.is_cuda or t.is_pinned() for t in (k_pages, v_pages, page_table))

    def check_seen(self) -> None:
        if not self.seen:
            for t, name in ((self.k_pages, "k_pages"), (self.v_pages, "v_pages"), (self.page_table, "page_table")):
                _seen(t, name)

    def check_weights(self, weights, name: str = "weights") -> int:
        """Row pitch of fp32 [batch, kv_heads, slots] weights."""
        if weights is None:
            return 0
        if weights.dim() != 3 or weights.shape[:2] != (self.batch, self.kv_heads):
            raise ValueError(f"{name} must be [batch, kv_heads, slots]")
        _array(weights, _F32, weights.numel(), name)
        return weights.shape[2]


class Handle:
    def __init__(self):
        h = C.c_void_p()
        check(lib.grxdnnCreate(C.byref(h)), "grxdnnCreate")
        self.h = h

    def close(self) -> int:
        if self.h:
            s = lib.grxdnnDestroy(self.h)
            self.h = None
            return s
        return N.SUCCESS

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_stream(self, stream) -> int:
        return lib.grxdnnSetStream(self.h, stream_ptr(stream))

    def execution_status(self) -> int:
        return lib.grxdnnGetExecutionStatus(self.h)

    def rmsnorm(self, x, gamma, eps, y, rstd=None, rows=None, hidden=None, ldx=None, ldy=None) -> int:
        rows = x.shape[0] if rows is None else rows
        hidden = x.shape[1] if hidden is None else hidden
        ldx = x.stride(0) if ldx is None else ldx
        ldy = y.stride(0) if ldy is None else ldy
        return lib.grxdnnRMSNormForward(self.h, rows, hidden, ptr(x), dtype_code(x), ldx, ptr(gamma), eps, ptr(y),
                                        dtype_code(y), ldy, ptr(rstd))

    def layernorm(self, x, gamma, beta, eps, y, mean=None, rstd=None, rows=None, hidden=None, ldx=None,
                  ldy=None) -> int:
        rows = x.shape[0] if rows is None else rows
        hidden = x.shape[1] if hidden is None else hidden
        ldx = x.stride(0) if ldx is None else ldx
        ldy = y.stride(0) if ldy is None else ldy
        return lib.grxdnnLayerNormForward(self.h, rows, hidden, ptr(x), dtype_code(x), ldx, ptr(gamma), ptr(beta),
                                          eps, ptr(y), dtype_code(y), ldy, ptr(mean), ptr(rstd))

    def rmsnorm_backward(self, dy, x, gamma, eps, dx, rstd=None, dgamma=None) -> int:
        """grxdnnRMSNormBackward on [rows, hidden] tensors with row pitches from strides."""
        rows, hidden = x.shape
        return lib.grxdnnRMSNormBackward(self.h, rows, hidden, ptr(dy), dtype_code(dy), dy.stride(0), ptr(x),
                                         dtype_code(x), x.stride(0), ptr(gamma), ptr(rstd), eps, ptr(dx),
                                         dtype_code(dx), dx.stride(0), ptr(dgamma))

    def layernorm_backward(self, dy, x, gamma, eps, dx, mean=None, rstd=None, dgamma=None, dbeta=None) -> int:
        """grxdnnLayerNormBackward on [rows, hidden] tensors with row pitches from strides."""
        rows, hidden = x.shape
        return lib.grxdnnLayerNormBackward(self.h, rows, hidden, ptr(dy), dtype_code(dy), dy.stride(0), ptr(x),
                                           dtype_code(x), x.stride(0), ptr(gamma), ptr(mean), ptr(rstd), eps,
                                           ptr(dx), dtype_code(dx), dx.stride(0), ptr(dgamma), ptr(dbeta))

    def softmax(self, x, y, rows=None, cols=None, ldx=None, ldy=None) -> int:
        rows = x.shape[0] if rows is None else rows
        cols = x.shape[1] if cols is None else cols
        ldx = x.stride(0) if ldx is None else ldx
        ldy = y.stride(0) if ldy is None else ldy
        return lib.grxdnnSoftmaxForward(self.h, rows, cols, ptr(x), dtype_code(x), ldx, ptr(y), dtype_code(y), ldy)

    def gelu(self, x, y, mode: int = 0, n=None) -> int:
        n = x.numel() if n is None else n
        return lib.grxdnnGeluForward(self.h, n, ptr(x), dtype_code(x), ptr(y), dtype_code(y), mode)

    def attention_backward(self, q, k, v, o, dout, lse, scale, causal, dq, dk, dv) -> int:
        """grxdnnAttentionBackward on [B, H, S, D] tensors (descriptors from strides)."""
        ds = [attn_desc(t) for t in (q, k, v, o, dout, dq, dk, dv)]
        return lib.grxdnnAttentionBackward(self.h, C.byref(ds[0]), ptr(q), C.byref(ds[1]), ptr(k), C.byref(ds[2]),
                                           ptr(v), C.byref(ds[3]), ptr(o), C.byref(ds[4]), ptr(dout), ptr(lse),
                                           scale, 1 if causal else 0, C.byref(ds[5]), ptr(dq), C.byref(ds[6]),
                                           ptr(dk), C.byref(ds[7]), ptr(dv))

    def conv2d(self, x, w, y, pad=(0, 0), stride=(1, 1), dilation=(1, 1), bias=None, activation=0, alpha=None,
               beta=None) -> int:
        """grxdnnConv2dForward: x [n, h, w, c] NHWC, w [k, r, s, c] KRSC, y [n, p, q, k]."""
        d = conv_desc(x, w, pad, stride, dilation)
        a = C.c_float(alpha) if alpha is not None else None
        b = C.c_float(beta) if beta is not None else None
        return lib.grxdnnConv2dForward(self.h, C.byref(d), ptr(x), dtype_code(x), ptr(w), dtype_code(w),
                                       C.byref(a) if a is not None else None, C.byref(b) if b is not None else None,
                                       ptr(bias), activation, ptr(y), dtype_code(y))

    def pool2d(self, x, y, window, pad=(0, 0), stride=None, mode=0) -> int:
        """grxdnnPooling2dForward on NHWC tensors."""
        d = pool_desc(x, window, pad, stride or window, mode)
        return lib.grxdnnPooling2dForward(self.h, C.byref(d), ptr(x), dtype_code(x), ptr(y), dtype_code(y))

    def softmax_backward(self, y, dy, dx) -> int:
        """grxdnnSoftmaxBackward on [rows, cols] tensors (row pitches from strides)."""
        rows, cols = y.shape
        return lib.grxdnnSoftmaxBackward(self.h, rows, cols, ptr(y), dtype_code(y), y.stride(0), ptr(dy),
                                         dtype_code(dy), dy.stride(0), ptr(dx), dtype_code(dx), dx.stride(0))

    def gelu_backward(self, x, dy, dx, mode: int = 0) -> int:
        """grxdnnGeluBackward over x.numel() contiguous elements."""
        return lib.grxdnnGeluBackward(self.h, x.numel(), ptr(x), ptr(dy), ptr(dx), dtype_code(x), mode)

    def attention(self, q, k, v, o, scale, causal, lse=None, descs=None) -> int:
        dq, dk, dv, do = descs if descs is not None else (attn_desc(q), attn_desc(k), attn_desc(v), attn_desc(o))
        return lib.grxdnnAttentionForward(self.h, C.byref(dq), ptr(q), C.byref(dk), ptr(k), C.byref(dv), ptr(v),
                                          C.byref(do), ptr(o), scale, 1 if causal else 0, ptr(lse))

    def kv_append(self, cache, lens, k, v, counts=None, lens_out=None) -> int:
        """grxdnnKvCacheAppend: k, v [batch, kv_heads, tokens, head_dim] enter `cache` at lens[b], of which the first
        counts[b] each (all of them without counts). lens_out (may be lens) receives the new lengths."""
        n = cache.batch
        if not cache.seen:
            cache.check_seen()
        return lib.grxdnnKvCacheAppend(self.h, cache.ref, cache.k, cache.v, cache.table, _array(lens, _I32, n, "lens"),
                                       _attn(k, "k"), k.data_ptr(), _attn(v, "v"), v.data_ptr(),
                                       _array(counts, _I32, n, "counts"), _array(lens_out, _I32, n, "lens_out"))

    def paged_attention(self, cache, lens, q, o, scale, window=0, lse=None, weights=None) -> int:
        """grxdnnPagedAttentionForward: q, o [batch, heads, 1, head_dim]; lse fp32 [batch, heads]; weights fp32
        [batch, kv_heads, slots >= cache.capacity], added to."""
        pitch = cache.check_weights(weights)
        if not cache.seen:
            cache.check_seen()
        return lib.grxdnnPagedAttentionForward(self.h, cache.ref, cache.k, cache.v, cache.table,
                                               _array(lens, _I32, cache.batch, "lens"), _attn(q, "q"), q.data_ptr(),
                                               _attn(o, "o"), o.data_ptr(), scale, window,
                                               None if lse is None else _array(lse, _F32, q.shape[0] * q.shape[1], "lse"),
                                               ptr(weights), pitch)

    def kv_evict(self, cache, lens, weights, keep, recent, out=None, lens_out=None, weights_out=None,
                 indices=None) -> int:
        """grxdnnKvCacheEvict into the cache `out` with its lengths and weights, or in place without them. indices:
        int32 [batch, kv_heads, keep]."""
        if (out is None) != (lens_out is None) or (out is None) != (weights_out is None):
            raise ValueError("out, lens_out and weights_out go together")
        if out is None:
            out, lens_out, weights_out = cache, lens, weights
        pitch, pitch_out = cache.check_weights(weights), out.check_weights(weights_out, "weights_out")
        cache.check_seen()
        out.check_seen()
        return lib.grxdnnKvCacheEvict(self.h, cache.ref, cache.k, cache.v, cache.table, _array(lens, _I32, cache.batch, "lens"),
                                      ptr(weights), pitch, keep, recent, out.ref, out.k, out.v, out.table,
                                      _array(lens_out, _I32, cache.batch, "lens_out"), ptr(weights_out), pitch_out,
                                      _array(indices, _I32, cache.batch * cache.kv_heads * keep, "indices"))

    def token_logprobs(self, logits, tokens, logp, scale=1.0, entropy=None, lse=None, top_tokens=None,
                       top_logp=None) -> int:
        """grxdnnTokenLogProbsForward on [rows, vocab] logits (row pitch from the stride); tokens int32 [rows];
        top_tokens int32 and top_logp fp32 [rows, k]."""
        code = dtype_code(logits)
        rows, vocab, ld = _rows(logits, "logits")
        top = top_tokens if top_tokens is not None else top_logp
        _, k = top.shape if top is not None else (rows, 0)
        return lib.grxdnnTokenLogProbsForward(self.h, rows, vocab, logits.data_ptr(), code, ld,
                                              scale, _array(tokens, _I32, rows, "tokens"),
                                              _array(logp, _F32, rows, "logp"), _array(entropy, _F32, rows, "entropy"),
                                              _array(lse, _F32, rows, "lse"), k,
                                              _array(top_tokens, _I32, rows * k, "top_tokens"),
                                              _array(top_logp, _F32, rows * k, "top_logp"))

    def token_logprobs_backward(self, logits, tokens, lse, dlogp, dlogits, scale=1.0, entropy=None,
                                dentropy=None) -> int:
        """grxdnnTokenLogProbsBackward: dlogits [rows, vocab] from dlogp and dentropy (fp32 [rows], either may be None)
        and the forward's lse and entropy. dlogits may be logits."""
        rows, vocab, ld = _rows(logits, "logits")
        drows, dvocab, ldd = _rows(dlogits, "dlogits")
        if (drows, dvocab) != (rows, vocab):
            raise ValueError("dlogits must have the shape of logits")
        code = dtype_code(logits)
        return lib.grxdnnTokenLogProbsBackward(self.h, rows, vocab, logits.data_ptr(), code, ld,
                                               scale, _array(tokens, _I32, rows, "tokens"), _array(lse, _F32, rows, "lse"),
                                               _array(entropy, _F32, rows, "entropy"),
                                               _array(dlogp, _F32, rows, "dlogp"),
                                               _array(dentropy, _F32, rows, "dentropy"), dlogits.data_ptr(),
                                               code if dlogits.dtype is logits.dtype else dtype_code(dlogits), ldd)
