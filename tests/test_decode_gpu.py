"""The decoding example, its operators run together: against a plain chain in 64 bits that rounds to bf16 where the
library stores bf16, with a cache that keeps everything and with one that evicts."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu
spec = importlib.util.spec_from_file_location("decode_example", Path(__file__).resolve().parent.parent / "examples" / "decode.py")
decode = importlib.util.module_from_spec(spec)
spec.loader.exec_module(decode)


def bf(x):
    return x.to(torch.bfloat16).double()


def plain_chain(m, tokens):
    """Hidden states after the last norm, of whole sequences [batch, n]."""
    batch, n = tokens.shape

    def norm(x):
        return bf(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5))

    x = m.embed[tokens.long()].double()
    mask = torch.full((n, n), -math.inf, device="cuda", dtype=torch.float64).triu(1)
    for w in m.blocks:
        q, k, v = bf(norm(x) @ w["qkv"].double().T).view(batch, n, 3, m.heads, m.dim).permute(2, 0, 3, 1, 4)
        p = torch.softmax(q @ k.transpose(2, 3) / math.sqrt(m.dim) + mask, -1)
        x = bf(x + bf((p @ v).transpose(1, 2).reshape(batch, n, -1)) @ w["o"].double().T)
        up = bf(torch.nn.functional.gelu(norm(x) @ w["up"].double().T, approximate="tanh"))
        x = bf(x + up @ w["down"].double().T)
    return norm(x)


def test_decoding_matches_a_plain_chain(dev):
    m = decode.Model()
    prompt = torch.randint(m.vocab, (3, 40), device="cuda", dtype=torch.int32)
    d = decode.Decoder(m, 3, budget=64, recent=8, room=65)  # 40 + 10 tokens: nothing is evicted
    answers, logp, entropy, alternatives, states = d.answer(prompt, 10)
    advantage = torch.randn(30, device="cuda")
    again, grad = d.learn(states.flatten(0, 1), answers.flatten().contiguous(), advantage)
    assert d.layers[0]["lens"].tolist() == [50] * 3
    d.close()
    hidden = plain_chain(m, torch.cat([prompt, answers], 1))[:, 39:49]
    # as the block's test: the chain's bf16 roundings fall together, what remains are ties of a rounding
    err = (states.double() - hidden).abs()
    assert (err <= 3e-2 + 3e-2 * hidden.abs()).all(), err.max()
    logits = (states.double() @ m.out.double().T).flatten(0, 1)
    lse, want, ent, top, top_logp = R.score(bf(logits), 1.0, answers.flatten(), 5)
    assert torch.equal(alternatives.flatten(0, 1)[:, 0], answers.flatten())
    # logits are stored in bf16: each may fall on either side of a rounding
    assert ((logp.flatten().double() - want).abs() <= 2.0 ** -7 * (1 + logits.abs().amax(1))).all()
    assert ((entropy.flatten().double() - ent).abs() <= 1e-2).all()
    assert torch.allclose(again, logp.flatten(), atol=1e-5)
    dx = R.score_grad(bf(logits), 1.0, answers.flatten(), -advantage, torch.full((30,), -0.01, device="cuda"))
    want = dx.T @ states.flatten(0, 1).double()
    assert (grad.double() - want).norm() <= 1e-2 * want.norm()


def test_decoding_with_a_bounded_cache(dev):
    m = decode.Model()
    prompt = torch.randint(m.vocab, (4, 60), device="cuda", dtype=torch.int32)
    d = decode.Decoder(m, 4, budget=48, recent=16, room=61)  # room for the prompt; 48 tokens are kept
    answers, logp, entropy, alternatives, _ = d.answer(prompt, 30)
    for layer in d.layers:
        assert layer["lens"].tolist() == [48] * 4
        w = layer["weights"]
        assert (w[..., :48] >= 0).all() and (w[..., 48:] == 0).all()
        # every step hands out a weight of 1 a query head, of which evicted keys took some along
        assert (w.sum(2) <= 30 * (1 + 1e-5)).all() and (w.sum(2) > 0).all()
    assert (logp <= 0).all() and (entropy >= 0).all() and torch.isfinite(logp).all()
    d.close()


def test_the_example_runs(dev, capsys):
    decode.main()
    assert "scored again" in capsys.readouterr().out
