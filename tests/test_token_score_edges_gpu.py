"""Scoring where 32 bits have little left after the point: rows and scales whose largest scaled logit is far from 0."""
import math

import pytest
import torch

import serving_ref as R
from grxcp_b200 import _native as N

pytestmark = pytest.mark.gpu
REL = 2.0 ** -16  # of lse and entropies at these sizes, as derived in test_token_score_gpu.py
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def scores(dnn, x, t, scale, entropy=True, top=5):
    rows = x.shape[0]
    f = dict(device="cuda", dtype=torch.float32)
    logp, lse, ent = (torch.full((rows,), math.nan, **f) for _ in range(3))
    tt, tl = torch.full((rows, top), -5, dtype=torch.int32, device="cuda"), torch.full((rows, top), math.nan, **f)
    assert dnn.token_logprobs(x, t, logp, scale, ent if entropy else None, lse, tt, tl) == N.SUCCESS
    return logp, lse, ent, tt, tl


def check_largest(dnn, x, scale):
    """The given token is one of the row's largest: scale x minus the largest is then exactly 0, and logp is minus the
    logarithm of the sum of exponentials, off by REL of 1 and of itself, whatever the size of lse. The entropy's bound is
    that of any row."""
    t = x.float().nan_to_num(-math.inf, math.inf, -math.inf).argmax(1).to(torch.int32)
    r_lse, r_logp, r_ent, r_tt, r_tl = R.score(x, scale, t, 5)
    for entropy in (True, False):
        logp, lse, ent, tt, tl = scores(dnn, x, t, scale, entropy)
        assert ((logp.double() - r_logp).abs() <= REL * (1 + r_logp.abs())).all(), (scale, entropy, logp, r_logp)
        assert ((tl[:, 0].double() - r_tl[:, 0]).abs() <= REL * (1 + r_logp.abs())).all()
        assert ((lse.double() - r_lse).abs() <= REL + 2.0 ** -22 * r_lse.abs()).all()
        assert torch.equal(tt.long(), r_tt)
        if entropy:
            assert ((ent.double() - r_ent).abs() <= REL * (2 + 2 * math.log(x.shape[1]) + 2 * r_ent)).all(), (scale, ent, r_ent)


@pytest.mark.parametrize("rows", [5, 700, 1500, 2500])  # clusters, four, two and one warp a row
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("largest", [1e6, 2.0 ** 24, 2.0 ** 27, 1.5e8, 1e9, 5e9, 8e9, 1e10, 1e12])
@pytest.mark.parametrize("sign", [1, -1])
def test_rows_far_from_zero(dnn, dtype, rows, largest, sign):
    """Logits that differ from the largest by a few of its last places, some equal to it, and -inf."""
    g = torch.Generator(device="cuda").manual_seed(1)
    top = torch.tensor(sign * largest, device="cuda").to(dtype).float()
    place = 2.0 ** (math.floor(math.log2(largest)) - (7 if dtype == torch.bfloat16 else 23))
    steps = torch.randint(0, 40, (rows, 2001), device="cuda", generator=g)
    x = (top.double() - place * steps).to(dtype)
    x[torch.rand(rows, 2001, device="cuda", generator=g) < 0.5] = -math.inf
    x[:, 100] = top.to(dtype)
    check_largest(dnn, x, 1.0)


@pytest.mark.parametrize("rows", [5, 700, 1500, 2500])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [1e4, 1e6, 1e7, 1e8, 1e9, 1e10])
def test_sharp_temperatures(dnn, dtype, rows, scale):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = (6 * torch.randn(rows, 3001, device="cuda", generator=g)).to(dtype)
    x[1::3, ::2] = -math.inf
    x[2::3] += 20.0
    check_largest(dnn, x, scale)


def check_given_lse(dnn, x, t, lse, ent, scale):
    """The formula at the given lse and entropy. p is off by REL of itself and, where the given lse is taken for the row's
    own, by the two last places of 32 bits in which the two may differ; x - lse is off by the same and 2^-23 of itself."""
    rows = x.shape[0]
    dlogp, dent = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    z, far = x.double() * scale, lse.double()[:, None]
    d = z - far
    p = torch.exp(d)
    hit = torch.zeros_like(d).scatter_(1, t.long()[:, None], 1.0)
    pd = torch.where(p == 0, torch.zeros_like(p), p * (d + ent.double()[:, None]))
    off = REL + 2.0 ** -22 * far.abs() * (far.abs() > 512)
    logs = torch.where(p == 0, torch.zeros_like(p), d.abs()) + ent.double()[:, None].abs()
    for g, h in ((dlogp, None), (None, dent), (dlogp, dent)):
        dx = torch.full_like(x, math.nan)
        assert dnn.token_logprobs_backward(x, None if g is None else t, lse, g, dx, scale, None if h is None else ent, h) == N.SUCCESS
        gl = torch.zeros(rows, 1, device="cuda", dtype=torch.float64) if g is None else g.double()[:, None]
        ge = torch.zeros_like(gl) if h is None else h.double()[:, None]
        want = scale * (gl * (hit - p) - ge * pd)
        u = R.ROUND.get(x.dtype, 2.0 ** -22)
        tol = u * want.abs() + scale * 4 * off * p * (gl.abs() + ge.abs() * (1 + logs)) + 2.0 ** -24
        assert ((dx.double() - want).abs() <= tol).all(), ((dx.double() - want).abs() - tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("middle", [-40_000.0, -3000.0, -520.0, -500.0, 0.0, 500.0, 520.0, 3000.0, 40_000.0])
@pytest.mark.parametrize("share", ["half", "most", "little", "none"])
def test_gradient_from_the_lse_of_a_whole_vocabulary(dnn, dtype, middle, share):
    """Logits are a part of a vocabulary; lse and entropy are the whole's."""
    g = torch.Generator(device="cuda").manual_seed(5)
    whole = (middle + 2 * torch.randn(6, 8000, device="cuda", generator=g)).to(dtype)
    x = whole[:, :4000].contiguous()
    whole[:, 4000:] += {"half": 0.0, "most": -4.0, "little": 4.0, "none": -math.inf}[share]
    x[1, ::3] = whole[1, :4000:3] = -math.inf
    t = torch.randint(4000, (6,), device="cuda", generator=g).to(torch.int32)
    lp, lse = R.log_softmax(whole.double())
    p = torch.exp(lp)
    ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1)
    check_given_lse(dnn, x, t, lse.float(), ent.float(), 1.0)


@pytest.mark.parametrize("rows", [5, 700, 1500, 2500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [1.5, 3.0, 1000.0])
def test_rows_whose_largest_passes_32_bits_once_scaled(dnn, dtype, rows, scale):
    """Rows of the type's lowest value and nothing above it, at a sharp temperature; one of its largest. What is left of
    them in logp, the entropy and the gradient has no infinity in it."""
    vocab, low = 1501, torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.full((rows, vocab), low, device="cuda", dtype=dtype)
    x[1::3, 100:] = -math.inf
    x[2::3] = torch.randn(x[2::3].shape, device="cuda", generator=g).to(dtype)
    x[2::3, 7] = -low
    t = torch.randint(100, (rows,), device="cuda", generator=g).to(torch.int32)
    t[2::3] = 7
    largest = torch.full((rows,), 1501, device="cuda", dtype=torch.float64)  # of them, a row
    largest[1::3], largest[2::3] = 100, 1
    want = -torch.log(largest)
    top = 1  # the rest of a row's order is that of 32 bits
    logp, lse, ent, tt, tl = scores(dnn, x, t, scale, top=top)
    plain, plain_lse, _, _, _ = scores(dnn, x, t, scale, entropy=False, top=top)
    tol = REL * (1 + want.abs())
    assert ((logp.double() - want).abs() <= tol).all() and ((plain.double() - want).abs() <= tol).all()
    assert ((tl[:, 0].double() - want).abs() <= tol).all()
    assert torch.equal(tt[:, 0], torch.where(largest == 1, 7, 0).to(torch.int32))
    assert ((ent.double() + want).abs() <= REL * (2 + 2 * math.log(vocab) + 2 * want.abs())).all()
    last = torch.finfo(torch.float32).max
    assert torch.equal(lse, torch.where(largest == 1, last, -last).float()) and torch.equal(plain_lse, lse)
    dlogp, dx = torch.randn(rows, device="cuda", generator=g), torch.full_like(x, math.nan)
    assert dnn.token_logprobs_backward(x, t, lse, dlogp, dx, scale, ent, torch.zeros(rows, device="cuda")) == N.SUCCESS
    p = torch.where(x == x.amax(1, keepdim=True), 1 / largest[:, None], torch.zeros(1, device="cuda", dtype=torch.float64))
    hit = torch.zeros_like(p).scatter_(1, t.long()[:, None], 1.0)
    grad = scale * dlogp.double()[:, None] * (hit - p)
    u = R.ROUND.get(dtype, 2.0 ** -22)
    assert ((dx.double() - grad).abs() <= u * grad.abs() + 4 * REL * scale * dlogp.double().abs()[:, None] * p + 2.0 ** -24).all()
