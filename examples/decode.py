"""Decoding with a bounded key-value cache, and learning from what was decoded, through the library alone.

A small pre-norm transformer with random weights reads a batch of prompts, then answers token by token:

    prompt    GemmEx projections, grxdnnAttentionForward (causal), grxdnnKvCacheAppend of all keys and values at once
    a token   GemmEx, grxdnnKvCacheAppend, grxdnnPagedAttentionForward (adding up what each key receives),
              grxdnnTokenLogProbsForward on the logits (the chosen token, its alternatives, the entropy),
              grxdnnKvCacheEvict once a cache holds more than its budget
    learning  grxdnnTokenLogProbsForward / Backward on the answers' logits, GemmEx for the output matrix's gradient

Lengths stay on the device: nothing here waits for the GPU between tokens. Usage: python examples/decode.py
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from grxcp_b200 import _native as N  # noqa: E402
from grxcp_b200 import blas as B  # noqa: E402
from grxcp_b200 import dnn as D  # noqa: E402

BF16 = torch.bfloat16


class Model:
    """Random weights; linear layers are [out, in], row-major."""

    def __init__(self, layers=2, hidden=512, heads=4, vocab=5003, seed=0):
        self.layers, self.hidden, self.heads, self.dim, self.vocab = layers, hidden, heads, 128, vocab
        g = torch.Generator(device="cuda").manual_seed(seed)
        inner = heads * self.dim

        def w(out, inp):
            return (torch.randn(out, inp, device="cuda", generator=g) / math.sqrt(inp)).to(BF16)

        self.embed = torch.randn(vocab, hidden, device="cuda", generator=g).to(BF16)
        self.blocks = [dict(qkv=w(3 * inner, hidden), o=w(hidden, inner), up=w(4 * hidden, hidden), down=w(hidden, 4 * hidden))
                       for _ in range(layers)]
        self.out = w(vocab, hidden)
        self.gamma = torch.ones(hidden, device="cuda")


class Decoder:
    """One batch of sequences: its caches, one per layer, and the library's handles."""

    def __init__(self, model, batch, budget, recent, room, page=16):
        self.m, self.batch, self.budget, self.recent = model, batch, budget, recent
        self.blas, self.dnn = B.Handle(), D.Handle()
        self.scale = 1 / math.sqrt(model.dim)
        pages = -(-room // page)
        self.layers = []
        for _ in range(model.layers):
            k, v = (torch.zeros(batch * pages, page, model.heads, model.dim, device="cuda", dtype=BF16) for _ in range(2))
            table = torch.randperm(batch * pages, device="cuda").to(torch.int32).reshape(batch, pages)
            cache = D.PagedCache(k, v, table)
            self.layers.append(dict(cache=cache, lens=torch.zeros(batch, device="cuda", dtype=torch.int32),
                                    weights=torch.zeros(batch, model.heads, cache.capacity, device="cuda")))

    def linear(self, x, w, out, beta=0.0, act=N.ACT_NONE):
        """out = act(x W^T) + beta out, on [tokens, features] tensors."""
        o, i = w.shape
        B.check(self.blas.set_epilogue(activation=act))
        B.check(self.blas.gemm_ex(N.OP_T, N.OP_N, o, x.shape[0], i, 1.0, w, N.GRX_R_16BF, i, x, N.GRX_R_16BF, i, beta, out,
                                  N.GRX_R_16BF, o))
        return out

    def norm(self, x):
        y = torch.empty_like(x)
        D.check(self.dnn.rmsnorm(x, self.m.gamma, 1e-5, y))
        return y

    def forward(self, tokens):
        """Hidden states [batch * n, hidden] of n more tokens of every sequence ([batch, n]); n > 1 only for the prompt."""
        m, (batch, n) = self.m, tokens.shape
        x = m.embed[tokens.flatten().long()]
        for block, layer in zip(m.blocks, self.layers):
            inner = m.heads * m.dim
            qkv = self.linear(self.norm(x), block["qkv"], torch.empty(batch * n, 3 * inner, device="cuda", dtype=BF16))
            q, k, v = qkv.view(batch, n, 3, m.heads, m.dim).permute(2, 0, 3, 1, 4)
            attn = torch.empty(batch, n, m.heads, m.dim, device="cuda", dtype=BF16)
            D.check(self.dnn.kv_append(layer["cache"], layer["lens"], k, v, None, layer["lens"]))
            if n > 1:
                D.check(self.dnn.attention(q, k, v, attn.transpose(1, 2), self.scale, True))
            else:
                D.check(self.dnn.paged_attention(layer["cache"], layer["lens"], q, attn.transpose(1, 2), self.scale,
                                                 weights=layer["weights"]))
            self.linear(attn.view(batch * n, inner), block["o"], x, beta=1.0)
            up = torch.empty(batch * n, 4 * m.hidden, device="cuda", dtype=BF16)
            self.linear(self.linear(self.norm(x), block["up"], up, act=N.ACT_GELU_TANH), block["down"], x, beta=1.0)
        return self.norm(x)

    def logits(self, hidden):
        return self.linear(hidden, self.m.out, torch.empty(hidden.shape[0], self.m.vocab, device="cuda", dtype=BF16))

    def evict(self):
        for layer in self.layers:
            D.check(self.dnn.kv_evict(layer["cache"], layer["lens"], layer["weights"], self.budget, self.recent))

    def answer(self, prompt, steps, top=5):
        """Greedy answers [batch, steps]; logp, entropy and alternatives of each chosen token; the hidden states they were
        chosen from."""
        batch, f32 = self.batch, dict(device="cuda", dtype=torch.float32)
        hidden = self.forward(prompt).view(batch, -1, self.m.hidden)[:, -1].contiguous()
        chosen, logps, entropies, alternatives, states = [], [], [], [], []
        for _ in range(steps):
            logits = self.logits(hidden)
            tokens = torch.empty(batch, top, device="cuda", dtype=torch.int32)
            logp, entropy = torch.empty(batch, top, **f32), torch.empty(batch, **f32)
            D.check(self.dnn.token_logprobs(logits, None, None, 1.0, entropy, None, tokens, logp))
            chosen.append(tokens[:, 0])
            logps.append(logp[:, 0])
            entropies.append(entropy)
            alternatives.append(tokens)
            states.append(hidden)
            hidden = self.forward(tokens[:, :1])
            self.evict()  # the cache is never larger than its budget plus one token
        return tuple(torch.stack(t, 1) for t in (chosen, logps, entropies, alternatives, states))

    def learn(self, states, tokens, advantage, entropy_weight=0.01):
        """logp of the given tokens and the gradient of -sum(advantage logp) - entropy_weight sum(entropy) along the
        output matrix: fp32 [vocab, hidden]."""
        n, f32 = states.shape[0], dict(device="cuda", dtype=torch.float32)
        logits = self.logits(states)
        logp, entropy, lse = (torch.empty(n, **f32) for _ in range(3))
        D.check(self.dnn.token_logprobs(logits, tokens, logp, 1.0, entropy, lse))
        D.check(self.dnn.token_logprobs_backward(logits, tokens, lse, -advantage, logits, 1.0, entropy,
                                                 torch.full_like(entropy, -entropy_weight)))
        grad = torch.empty(self.m.vocab, self.m.hidden, **f32)
        B.check(self.blas.set_epilogue())
        # [hidden, vocab] column by column: states^T (as stored) times the logits' gradient
        B.check(self.blas.gemm_ex(N.OP_N, N.OP_T, self.m.hidden, self.m.vocab, n, 1.0, states, N.GRX_R_16BF, self.m.hidden,
                                  logits, N.GRX_R_16BF, self.m.vocab, 0.0, grad, N.GRX_R_32F, self.m.hidden))
        return logp, grad

    def close(self):
        B.check(self.blas.execution_status())
        D.check(self.dnn.execution_status())
        self.blas.close()
        self.dnn.close()


def main() -> None:
    model = Model()
    batch, prompt_len, steps, budget = 8, 96, 64, 112
    prompt = torch.randint(model.vocab, (batch, prompt_len), device="cuda", dtype=torch.int32)
    decoder = Decoder(model, batch, budget, recent=32, room=budget + 1)
    answers, logp, entropy, alternatives, states = decoder.answer(prompt, steps)
    advantage = torch.randn(batch * steps, device="cuda")
    again, grad = decoder.learn(states.flatten(0, 1), answers.flatten().contiguous(), advantage)
    decoder_lens = decoder.layers[0]["lens"].tolist()
    decoder.close()
    print(f"{batch} prompts of {prompt_len} tokens, {steps} tokens each; caches hold {decoder_lens} of {prompt_len + steps} tokens")
    print(f"first answer: {answers[0, :8].tolist()} ...  logp {logp[0, 0]:.3f}  entropy {entropy[0, 0]:.3f}  "
          f"alternatives {alternatives[0, 0].tolist()}")
    print(f"scored again: largest difference of logp {(again - logp.flatten()).abs().max():.2e}; "
          f"gradient of the output matrix: norm {grad.norm():.3f}")


if __name__ == "__main__":
    main()
