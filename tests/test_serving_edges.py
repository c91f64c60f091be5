"""CPU checks of the serving entry points at the edges of what they take: refused before any device is touched."""
import ctypes as C

import pytest

from grxcp_b200 import _native as N
from grxcp_b200 import dnn as D

P = 1 << 20  # any aligned non-null address: validation returns before it is touched
L = N.lib


@pytest.fixture()
def h():
    with D.Handle() as hh:
        yield hh.h


def cache(batch=2, kv_heads=4, dim=128, pages=10, page=16, width=5):
    return N.grxdnnPagedCache_t(batch, kv_heads, dim, pages, page, width, width, page * kv_heads * dim, kv_heads * dim, dim, N.GRX_R_16BF)


def evict(h, c, o, w, pitch, wo, pitch_out, keep=32):
    return L.grxdnnKvCacheEvict(h, C.byref(c), P, P, P, P, w, pitch, keep, 4, C.byref(o), 2 * P, 2 * P, 2 * P, 2 * P, wo, pitch_out, None)


def test_weights_over_themselves_need_one_pitch(h):
    """Rows of one pitch over rows of another would lie on other heads' weights."""
    assert evict(h, cache(), cache(), P, 80, P, 81) == N.INVALID_VALUE
    assert evict(h, cache(), cache(), P, 96, P, 80) == N.INVALID_VALUE


def test_addresses_between_elements(h):
    """A value's address that is no multiple of its size would be a misaligned access on the GPU."""
    c, q, kv, r = cache(), D.attn_desc(None, 2, 8, 1, 128), D.attn_desc(None, 2, 4, 1, 128), C.byref

    def refused(call, args, which):
        for i in which:
            for off in (1, 2, 3):
                assert call(*[P + off if j == i else a for j, a in enumerate(args)]) == N.INVALID_VALUE, (call.__name__, i, off)

    refused(L.grxdnnKvCacheAppend, [h, r(c), P, P, P, P, r(kv), P, r(kv), P, P, P], (4, 5, 10, 11))
    refused(L.grxdnnPagedAttentionForward, [h, r(c), P, P, P, P, r(q), P, r(q), P, 0.1, 0, P, P, 80], (4, 5, 12, 13))
    refused(L.grxdnnKvCacheEvict, [h, r(c), P, P, P, P, P, 80, 32, 4, r(c), P, P, P, P, 2 * P, 80, P], (4, 5, 6, 13, 14, 15, 17))
    scores = [h, 4, 1000, P, N.GRX_R_32F, 1000, 1.0, P, P, P, P, 5, P, P]
    refused(L.grxdnnTokenLogProbsForward, scores, (3, 7, 8, 9, 10, 12, 13))
    grad = [h, 4, 1000, P, N.GRX_R_32F, 1000, 1.0, P, P, P, P, P, 2 * P, N.GRX_R_32F, 1000]
    refused(L.grxdnnTokenLogProbsBackward, grad, (3, 7, 8, 9, 10, 11, 12))
    for type_ in (N.GRX_R_16BF, N.GRX_R_16F):
        for off in (1, 3):
            assert L.grxdnnTokenLogProbsForward(h, 4, 1000, P + off, type_, 1000, 1.0, P, P, P, P, 0, None, None) == N.INVALID_VALUE
            for x, dx in ((P + off, 2 * P), (P, 2 * P + off)):
                assert L.grxdnnTokenLogProbsBackward(h, 4, 1000, x, type_, 1000, 1.0, P, P, P, P, P, dx, type_, 1000) == N.INVALID_VALUE


MOST = 2 ** 31 - 1 - 2 ** 20


def test_counts_near_the_end_of_32_bits(h):
    """Loops over slots, tokens and heads step past their end by up to a grid's reach: what would pass 2^31 - 1 on the way,
    and go on at negative offsets, is refused."""
    def attention(c, heads=8):
        q = D.attn_desc(None, c.batch, heads, 1, c.headDim)
        return L.grxdnnPagedAttentionForward(h, C.byref(c), P, P, P, P, C.byref(q), P, C.byref(q), P, 0.1, 0, None, None, 0)

    def append(c):
        kv = D.attn_desc(None, c.batch, c.kvHeads, 1, c.headDim)
        return L.grxdnnKvCacheAppend(h, C.byref(c), P, P, P, P, C.byref(kv), P, C.byref(kv), P, None, None)

    for page, width in ((1, MOST + 1), (2 ** 31 - 1, 1), (16, 2 ** 27 - 1), (3, (2 ** 31 - 1) // 3)):
        assert MOST < page * width < 2 ** 31
        c = cache(page=page, width=width)
        assert append(c) == N.NOT_SUPPORTED and attention(c) == N.NOT_SUPPORTED
        assert evict(h, c, cache(), P, 1 << 33, 2 * P, 80) == N.NOT_SUPPORTED
        assert evict(h, cache(), c, P, 80, 2 * P, 1 << 33) == N.NOT_SUPPORTED
    heads = MOST // 64 + 1
    assert append(cache(kv_heads=heads, dim=64)) == N.NOT_SUPPORTED
    assert attention(cache(batch=1, kv_heads=1, dim=64), heads) == N.NOT_SUPPORTED
    assert append(cache(batch=MOST + 1, kv_heads=1)) == N.NOT_SUPPORTED


class OnGpu:
    """Tensors that stand in for tensors on the GPU: their memory is the host's, and no call may reach the library."""

    def __init__(self):
        import torch

        class Tensor(torch.Tensor):
            is_cuda = True
        self.kind = Tensor

    def __call__(self, *shape, dtype=None):
        import torch
        return torch.zeros(*shape, dtype=dtype).as_subclass(self.kind)


def test_tensors_in_host_memory_are_refused():
    """Each argument's turn."""
    import torch

    gpu, bf, i32 = OnGpu(), torch.bfloat16, torch.int32
    k, table = gpu(6, 16, 2, 64, dtype=bf), gpu(3, 2, dtype=i32)
    good = D.PagedCache(k, k, table)
    bad = [D.PagedCache(k.as_subclass(torch.Tensor), k, table), D.PagedCache(k, k.as_subclass(torch.Tensor), table),
           D.PagedCache(k, k, table.as_subclass(torch.Tensor))]
    lens, q, w = gpu(3, dtype=i32), gpu(3, 2, 1, 64, dtype=bf), gpu(3, 2, 32)
    x, t, f, tt, tl = gpu(4, 10), gpu(4, dtype=i32), gpu(4), gpu(4, 2, dtype=i32), gpu(4, 2)
    calls = {
        "kv_append": dict(cache=good, lens=lens, k=q, v=q.clone(), counts=lens.clone(), lens_out=lens.clone()),
        "paged_attention": dict(cache=good, lens=lens, q=q, o=q.clone(), scale=0.1, lse=gpu(3, 2), weights=w),
        "kv_evict": dict(cache=good, lens=lens, weights=w, keep=4, recent=1, out=good, lens_out=lens.clone(), weights_out=w.clone(),
                         indices=gpu(3, 2, 4, dtype=i32)),
        "token_logprobs": dict(logits=x, tokens=t, logp=f, entropy=f.clone(), lse=f.clone(), top_tokens=tt, top_logp=tl),
        "token_logprobs_backward": dict(logits=x, tokens=t, lse=f, dlogp=f.clone(), dlogits=x.clone(), entropy=f.clone(), dentropy=f.clone()),
    }
    with D.Handle() as hh:
        handle, hh.h = hh.h, None  # without a handle the library answers at once, whatever else it is given
        try:
            for name, args in calls.items():
                assert getattr(hh, name)(**args) == N.NOT_INITIALIZED, name
                for key, value in args.items():
                    if isinstance(value, torch.Tensor):
                        with pytest.raises(ValueError, match=f"^{key} must be on the GPU"):
                            getattr(hh, name)(**{**args, key: value.as_subclass(torch.Tensor)})
                    elif isinstance(value, D.PagedCache):
                        for other, part in zip(bad, ("k_pages", "v_pages", "page_table")):
                            with pytest.raises(ValueError, match=f"^{part} must be on the GPU"):
                                getattr(hh, name)(**{**args, key: other})
        finally:
            hh.h = handle


def test_kernels_that_start_early_use_no_read_only_loads():
    """A serving kernel may begin before the one that writes its lengths or pages has ended. The read-only path promises
    that what it reads does not change from the kernel's beginning on, so a load through it could be moved before the
    wait, or find an old line."""
    import re
    from pathlib import Path

    csrc = Path(__file__).resolve().parent.parent / "grxcp_b200" / "csrc"
    for name in ("serving.cuh", "kv_cache.cu", "paged_attention.cu", "token_score.cu"):
        code = re.sub(r"//[^\n]*", "", (csrc / name).read_text())
        assert not re.search(r"__ldg\b|ld\.global\.nc|__restrict__", code), name


def test_tensors_of_other_types_and_shapes_are_refused_on_the_gpu_too():
    """The type, shape and order that the raw calls would misread, with nothing else to refuse."""
    import torch

    gpu, bf, i32 = OnGpu(), torch.bfloat16, torch.int32
    k = gpu(6, 16, 2, 64, dtype=bf)
    c = D.PagedCache(k, k, gpu(3, 2, dtype=i32))
    lens, q, w = gpu(3, dtype=i32), gpu(3, 4, 1, 64, dtype=bf), gpu(3, 2, 32)
    x, t, f = gpu(4, 10), gpu(4, dtype=i32), gpu(4)
    wrong = [(gpu(3, dtype=torch.int64), "lens"), (gpu(2, dtype=i32), "lens"), (gpu(6, dtype=i32)[::2], "lens")]
    with D.Handle() as hh:
        handle, hh.h = hh.h, None
        try:
            calls = [(hh.paged_attention, (c, bad, q, q, 0.1), {}, name) for bad, name in wrong]
            calls += [(hh.kv_append, (c, lens, q[:, :2], q[:, :2]), dict(counts=bad), "counts") for bad, _ in wrong]
            calls += [(hh.kv_append, (c, lens, q[:, :2], q[:, :2]), dict(lens_out=bad), "lens_out") for bad, _ in wrong]
            calls.append((hh.paged_attention, (c, lens, q, q, 0.1), dict(lse=gpu(3, 3)), "lse"))
            for bad in (gpu(3, 2, 32, dtype=torch.float64), gpu(3, 1, 32), gpu(3, 2, 64)[..., ::2], gpu(2, 32)):
                calls.append((hh.paged_attention, (c, lens, q, q, 0.1), dict(weights=bad), "weights"))
                calls.append((hh.kv_evict, (c, lens, bad, 4, 1), {}, "weights"))
            calls.append((hh.kv_evict, (c, lens, w, 4, 1), dict(indices=gpu(3, 2, 5, dtype=i32)), "indices"))
            for bad, name in ((dict(tokens=gpu(4, dtype=torch.int64)), "tokens"), (dict(logp=gpu(4, dtype=torch.float64)), "logp"),
                              (dict(logp=gpu(3)), "logp"), (dict(logits=gpu(10, 4).T), "logits"),
                              (dict(top_tokens=gpu(4, 2, dtype=i32), top_logp=gpu(4, 3)), "top_logp")):
                calls.append((hh.token_logprobs, (), {**dict(logits=x, tokens=t, logp=f), **bad}, name))
            calls.append((hh.token_logprobs_backward, (x, t, f, f, gpu(4, 9)), {}, "dlogits"))
            for call, args, more, name in calls:
                with pytest.raises(ValueError, match=f"^{name} ") as e:
                    call(*args, **more)
                assert "on the GPU" not in str(e.value), e.value
        finally:
            hh.h = handle
