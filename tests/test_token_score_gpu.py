"""Log probabilities, entropy and top alternatives of given tokens, and their gradient, against 64-bit forms.

Bounds: x = scale * logit is rounded once (2^-24 |x|), the largest is subtracted exactly or rounded once more, so an
exponential is off by at most (2 + 2 * 40) 2^-23 of itself where it matters (|x - max| < 40 before it vanishes), sums
add 2^-18 at these sizes; lse then by REL = 2^-16 at most plus 2^-22 |lse|. An entropy is a difference of
two numbers up to log(vocab) + its own size, each off by REL of itself and of the mean distance from the largest."""
import math

import pytest
import torch

import serving_ref as R
from grxcp_b200 import _native as N

pytestmark = pytest.mark.gpu
REL = 2.0 ** -16
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def logits_of(rows, vocab, dtype, seed=0, spread=3.0, pitch=None, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.full((rows, (pitch or vocab) + offset), math.nan, device="cuda", dtype=dtype)
    x = base[:, offset:offset + vocab]
    x.copy_(spread * torch.randn(rows, vocab, device="cuda", generator=g))
    t = torch.randint(vocab, (rows,), device="cuda", generator=g).to(torch.int32)
    return x, t


def check(dnn, x, t, scale=1.0, top=5):
    rows, vocab = x.shape
    f = dict(device="cuda", dtype=torch.float32)
    logp, lse, ent = (torch.full((rows,), math.nan, **f) for _ in range(3))
    tt = torch.full((rows, top), -5, dtype=torch.int32, device="cuda") if top else None
    tl = torch.full((rows, top), math.nan, **f) if top else None
    assert dnn.token_logprobs(x, t, logp, scale, ent, lse, tt, tl) == N.SUCCESS
    torch.cuda.synchronize()
    r_lse, r_logp, r_ent, r_tt, r_tl = R.score(x, scale, t, top)

    def close(got, want, tol, what):
        got = got.double()
        same = (got == want) | ((got - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want))
        assert same.all(), (what, got[~same][:4], want[~same][:4])
    close(lse, r_lse, REL + 2.0 ** -22 * r_lse.abs().nan_to_num(0, 0, 0), "lse")
    close(logp, r_logp, REL + 2.0 ** -21 * (r_logp.abs() + r_lse.abs()).nan_to_num(0, 0, 0), "logp")
    close(ent, r_ent, REL * (2 + 2 * math.log(vocab) + 2 * r_ent), "entropy")
    if top:
        assert torch.equal(tt.long(), r_tt)
        close(tl, r_tl, REL + 2.0 ** -21 * (r_tl.abs() + r_lse.abs()[:, None]).nan_to_num(0, 0, 0), "top_logp")
    return logp, lse, ent


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 31, 31), (2, 257, 32), (7, 1000, 5), (1, 32_000, 20), (300, 4099, 5),
                                            (9, 50_257, 32), (2, 131_072, 20), (40, 100_003, 1), (1, 300_001, 7), (17, 65_536, 0)])
def test_score_sizes(dnn, dtype, rows, vocab, top):
    x, t = logits_of(rows, vocab, dtype)
    check(dnn, x, t, 1.0, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pitch,offset", [(5003, 0), (5008, 1), (5001, 3), (6000, 8)])
def test_score_pitch_and_alignment(dnn, dtype, pitch, offset):
    x, t = logits_of(11, 5000, dtype, pitch=pitch, offset=offset)
    check(dnn, x, t, 0.8, 20)


@pytest.mark.parametrize("scale", [0.05, 0.7, 1.0, 3.0])
def test_score_scale_and_spread(dnn, scale):
    for spread in (0.0, 0.01, 1.0, 12.0):
        for dtype in TYPES:
            x, t = logits_of(6, 9001, dtype, spread=spread)
            check(dnn, x, t, scale, 20)


@pytest.mark.parametrize("dtype", TYPES)
def test_score_ties_and_order(dnn, dtype):
    """Equal logits in long runs, rows that rise and fall, top entries packed together or at the ends."""
    vocab = 20_000
    i = torch.arange(vocab, device="cuda")
    rows = torch.stack([torch.zeros(vocab, device="cuda"), (i % 7).float(), i.float() / 64, -i.float() / 64, (i // 4000).float(),
                        torch.where(i >= vocab - 32, 5.0, 0.0), torch.where(i < 32, 5.0, 0.0), torch.where(i % 16 == 3, -0.0, 0.0)])
    t = torch.randint(vocab, (8,), device="cuda").to(torch.int32)
    for top in (1, 20, 32):
        check(dnn, rows.to(dtype), t, 1.0, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [33, 5000, 70_000])
def test_score_masked(dnn, dtype, vocab):
    """-inf for most, all but one, all; the type's lowest value; NaN; tokens outside the vocabulary."""
    x, t = logits_of(9, vocab, dtype)
    x[0, torch.rand(vocab, device="cuda") < 0.99] = -math.inf
    x[1] = -math.inf
    x[1, vocab // 2] = 2.0
    x[2] = -math.inf
    x[3] = torch.finfo(dtype).min
    x[4, ::2] = torch.finfo(dtype).min
    x[5, vocab // 3] = math.nan
    x[6] = math.nan
    t[7], t[8] = -1, vocab
    t[0], t[1] = vocab - 1, vocab // 2
    logp, lse, ent = check(dnn, x, t, 1.0, 20)
    assert logp[2] == -math.inf and lse[2] == -math.inf and ent[2] == 0
    assert logp[7] == 0 and logp[8] == 0 and ent[1] == 0


def test_score_parts_of_its_outputs(dnn):
    x, t = logits_of(5, 3001, torch.bfloat16)
    full = check(dnn, x, t, 1.0, 4)
    f = dict(device="cuda", dtype=torch.float32)
    logp, lse, ent = (torch.empty(5, **f) for _ in range(3))
    tt, tl = torch.empty(5, 4, device="cuda", dtype=torch.int32), torch.empty(5, 4, **f)
    assert dnn.token_logprobs(x, t, logp) == N.SUCCESS
    assert dnn.token_logprobs(x, None, None, lse=lse) == N.SUCCESS
    assert dnn.token_logprobs(x, None, None, entropy=ent) == N.SUCCESS
    assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-5) for a, b in zip((logp, lse, ent), full))
    assert dnn.token_logprobs(x, None, None, top_tokens=tt) == N.SUCCESS
    assert dnn.token_logprobs(x, None, None, top_logp=tl) == N.SUCCESS
    want = R.score(x, 1.0, t, 4)
    assert torch.equal(tt.long(), want[3]) and torch.allclose(tl.double(), want[4], atol=1e-4)


def test_rows_past_32_bits_and_many_rows(dnn):
    rows, vocab = 70_001, 33_000
    x = torch.empty(rows, vocab, device="cuda", dtype=torch.bfloat16).normal_()
    t = torch.randint(vocab, (rows,), device="cuda").to(torch.int32)
    logp, lse = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    assert dnn.token_logprobs(x, t, logp, lse=lse) == N.SUCCESS
    for r in (0, 1, 65_076, rows - 1):
        want = torch.log_softmax(x[r].double(), 0)[t[r].long()]
        assert abs(logp[r].item() - want.item()) < 1e-4
    dlogp = torch.randn(rows, device="cuda")
    last = x[-1].clone()
    assert dnn.token_logprobs_backward(x, t, lse, dlogp, x) == N.SUCCESS  # in place
    want = R.score_grad(last[None], 1.0, t[-1:], dlogp[-1:], torch.zeros(1, device="cuda"))
    assert ((x[-1:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()


# ---------------------------------------------------------------- gradient

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (5, 1000), (2, 32_000), (130, 4099), (4, 131_072)])
@pytest.mark.parametrize("which", ["logp", "entropy", "both"])
def test_grad(dnn, dtype, rows, vocab, which):
    x, t = logits_of(rows, vocab, dtype, pitch=vocab + (vocab % 2), offset=1)
    if rows > 2:
        x[1, :-1] = -math.inf
        x[2] = -math.inf
        t[1] = vocab - 1
        t[0] = -1
    grad(dnn, x, t, 0.9, which)
    grad(dnn, x.contiguous(), t, 1.0, which)


def grad(dnn, x, t, scale, which):
    rows = x.shape[0]
    lse, ent, logp = (torch.empty(rows, device="cuda") for _ in range(3))
    assert dnn.token_logprobs(x, t, logp, scale, ent, lse) == N.SUCCESS
    dlogp = torch.randn(rows, device="cuda") if which != "entropy" else None
    dent = torch.randn(rows, device="cuda") if which != "logp" else None
    zero = torch.zeros(rows, device="cuda")
    dx = torch.full_like(x, math.nan)
    assert dnn.token_logprobs_backward(x, t if dlogp is not None else None, lse, dlogp, dx, scale, ent if dent is not None else None,
                                       dent) == N.SUCCESS
    want = R.score_grad(x, scale, t, zero if dlogp is None else dlogp, zero if dent is None else dent)
    # p is off by REL + 2^-22 |lse| of itself (the forward's bound of lse), the entropy by REL (2 + 2 log vocab + 2 H),
    # the result is rounded once
    lp = R.log_softmax(x.double() * scale)[0]
    p = torch.exp(lp)
    logs = torch.where(p > 0, lp.abs(), torch.zeros_like(lp))
    size = 2 * math.log(max(2, x.shape[1])) + 4
    part = p * ((0 if dlogp is None else dlogp.abs().double()[:, None]) + (0 if dent is None else dent.abs().double()[:, None]) * (logs + 3 * size))
    u = R.ROUND.get(x.dtype, 2.0 ** -22)
    tol = u * want.abs() + scale * 4 * REL * part + 2.0 ** -24
    assert ((dx.double() - want).abs() <= tol).all(), ((dx.double() - want).abs() - tol).max()


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_far_from_zero(dnn, dtype):
    """Rows whose lse has few digits left after the point: all of them at the type's lowest value, or moved far out."""
    x, t = logits_of(6, 3000, dtype)
    x[0] = torch.finfo(dtype).min
    x[1, ::2] = torch.finfo(dtype).min
    x[2] = -20_000.0
    x[3] = (x[3].float() * 300).to(dtype) + 30_000
    x[4] += 700.0
    for which in ("logp", "entropy", "both"):
        grad(dnn, x, t, 1.0, which)


def test_grad_against_differences(dnn):
    """The forward's own values at logits moved by h: a difference over 2 h is off by h^2 / 6 of a third derivative that
    a softmax keeps below 1 (entropy: below 8), and by twice the forward's bound over 2 h."""
    rows, vocab, h, scale = 4, 24, 2.0 ** -5, 1.1
    x, t = logits_of(rows, vocab, torch.float32, spread=1.5)
    dlogp, dent = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")

    def value(y):
        n = y.shape[0]
        logp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        assert dnn.token_logprobs(y, t.repeat(n // rows), logp, scale, ent) == N.SUCCESS
        return logp.double() * dlogp.double().repeat(n // rows) + ent.double() * dent.double().repeat(n // rows)

    lse, ent, logp = (torch.empty(rows, device="cuda") for _ in range(3))
    assert dnn.token_logprobs(x, t, logp, scale, ent, lse) == N.SUCCESS
    dx = torch.empty_like(x)
    assert dnn.token_logprobs_backward(x, t, lse, dlogp, dx, scale, ent, dent) == N.SUCCESS
    step = h * torch.eye(vocab, device="cuda")[:, None]
    up, down = value((x + step).flatten(0, 1)), value((x - step).flatten(0, 1))
    slope = ((up - down) / (2 * h)).reshape(vocab, rows).T
    size = dlogp.abs() + 8 * dent.abs()
    tol = (h * h / 6 * scale ** 3 + 2.0 ** -16 / h) * size.double()[:, None]
    assert ((dx.double() - slope).abs() <= tol).all()


def test_grad_in_place_equals_out_of_place(dnn):
    x, t = logits_of(33, 7777, torch.bfloat16)
    lse, logp = torch.empty(33, device="cuda"), torch.empty(33, device="cuda")
    assert dnn.token_logprobs(x, t, logp, lse=lse) == N.SUCCESS
    d = torch.randn(33, device="cuda")
    dx = torch.empty_like(x)
    assert dnn.token_logprobs_backward(x, t, lse, d, dx) == N.SUCCESS
    assert dnn.token_logprobs_backward(x, t, lse, d, x) == N.SUCCESS
    assert torch.equal(x, dx)


def test_score_on_a_side_stream(dnn):
    x, t = logits_of(64, 50_001, torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    dnn.set_stream(s)
    with torch.cuda.stream(s):
        check(dnn, x, t, 1.0, 20)
    dnn.set_stream(None)


@pytest.mark.parametrize("rows", [3, 600, 1300])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_score_orders_that_pass_every_bound(dnn, rows, top):
    """Rising rows, and runs of equal values that grow: almost every element is among the best so far."""
    vocab = 9001
    i = torch.arange(vocab, device="cuda").float()
    x = torch.stack([i / 32, (i / 700).floor(), -(i / 700).floor(), i % 977, torch.full_like(i, 3.0)]).repeat(rows // 5 + 1, 1)[:rows]
    t = torch.randint(vocab, (rows,), device="cuda").to(torch.int32)
    check(dnn, x.to(torch.bfloat16), t, 1.0, top)
    check(dnn, x, t, 0.7, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [200, 700, 1500])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
def test_score_many_rows(dnn, dtype, top, rows):
    x, t = logits_of(rows, 12_345, dtype, pitch=12_345, offset=0)
    x[::7, torch.rand(12_345, device="cuda") < 0.999] = -math.inf
    x[3::50] = -math.inf
    x[4::50, 100:] = math.nan
    check(dnn, x, t, 1.3, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(2400, 6_001), (4500, 3_003), (9000, 1_027)])
@pytest.mark.parametrize("top", [0, 1, 5, 9, 17, 32])
def test_score_a_warp_per_row(dnn, dtype, top, rows, vocab):
    x, t = logits_of(rows, vocab, dtype, pitch=vocab, offset=0)
    x[::7, torch.rand(vocab, device="cuda") < 0.99] = -math.inf
    x[3::50] = -math.inf
    x[4::50, 100:] = math.nan
    check(dnn, x, t, 1.3, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 400, 1000, 1500, 2500])
@pytest.mark.parametrize("top", [1, 7, 16, 32])
def test_score_orders(dnn, dtype, top, rows):
    vocab = 9_999
    x, t = logits_of(rows, vocab, dtype)
    ramp = torch.linspace(-8, 8, vocab, device="cuda")
    x[::5] = ramp.to(dtype)  # each part above all before it; in 16 bits with many equal neighbours
    x[1::5] = ramp.flip(0).to(dtype)
    x[2::5] = 1.5
    x[3::5] = (ramp + 4 * torch.sin(torch.arange(vocab, device="cuda") * 0.37)).to(dtype)
    check(dnn, x, t, 0.9, top)
