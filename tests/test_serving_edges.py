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
