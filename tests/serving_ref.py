"""Plain 64-bit forms of the token-serving operators, and the caches their tests run on."""
import math

import numpy as np
import torch

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # unit roundoff


def make_cache(lens, room, heads, dim, page, dtype, heads_first=False, seed=0, poison=True, spare=3):
    """K and V pools [pages, page, heads, dim], a table with room for `room` tokens in every row, and the sequences'
    tokens [n, heads, dim]. Pages lie in no order; table entries without tokens are -1; slots without tokens hold NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-room // page)) for _ in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).tolist()
    fill = math.nan if poison else 0.0
    k = torch.full((total, page, heads, dim), fill, dtype=dtype)
    v = torch.full((total, page, heads, dim), fill, dtype=dtype)
    width = max(max(need), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    tokens = []
    for b, n in enumerate(lens):
        row = [order.pop() for _ in range(need[b])]
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        kb = torch.randn(n, heads, dim, generator=g).to(dtype)
        vb = (torch.randn(n, heads, dim, generator=g) + 0.25).to(dtype)
        for i in range(n):
            k[row[i // page], i % page] = kb[i]
            v[row[i // page], i % page] = vb[i]
        tokens.append((kb, vb))
    k, v, table = k.cuda(), v.cuda(), table.cuda()
    if heads_first:
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    return k, v, table, tokens


def attention(tokens, q, scale, window, dtype):
    """o, lse, weights (lists by sequence) and the bounds of their rounding errors, in 64 bits.

    Rounding, u the type's unit roundoff: a score is a dot product of dim exact products summed in fp32 in some order,
    off by at most eps = (dim + 4) 2^-23 scale sum |q k|; it moves p by 2 eps of itself (numerator and total), the
    exponential and the sums by less than 2^-16 more. p may be rounded to the type before it meets V (u p |v|), the
    output is rounded once (u |o|)."""
    out = []
    for (k, v), qb in zip(tokens, q):
        n = k.shape[0]
        first = max(0, n - window) if window else 0
        k, v = k[first:].double(), v[first:].double()
        heads, dim = qb.shape
        group = heads // k.shape[1]
        if n == first:
            z = torch.zeros(heads, dim, dtype=torch.float64)
            out.append(dict(o=z, o_tol=z, lse=torch.full((heads,), -math.inf, dtype=torch.float64),
                            lse_tol=torch.zeros(heads, dtype=torch.float64), first=first,
                            w=torch.zeros(k.shape[1], 0, dtype=torch.float64), w_tol=torch.zeros(k.shape[1], 0, dtype=torch.float64)))
            continue
        kk, vv = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
        s = torch.einsum("hd,hnd->hn", qb.double(), kk) * scale
        eps = (dim + 4) * 2.0 ** -23 * scale * torch.einsum("hd,hnd->hn", qb.double().abs(), kk.abs()).amax(1)
        lse = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[:, None])
        o = torch.einsum("hn,hnd->hd", p, vv)
        u, rel = ROUND[dtype], 2 * eps + 2.0 ** -16
        pv = torch.einsum("hn,hnd->hd", p, vv.abs())
        out.append(dict(o=o, o_tol=u * o.abs() + (u + rel)[:, None] * pv + 2.0 ** -24, lse=lse,
                        lse_tol=eps + 2.0 ** -16 + 2.0 ** -22 * lse.abs(), first=first, w=p.unflatten(0, (-1, group)).sum(1),
                        w_tol=(p * rel[:, None]).unflatten(0, (-1, group)).sum(1) + 2.0 ** -23))
    return out


def evict(w, n, keep, recent):
    """Slots that one head keeps of n, by its weights (numpy fp32)."""
    if n <= keep:
        return list(range(n))
    age = n - min(n, recent)
    x = np.where(np.isnan(w[:age]), -np.inf, w[:age]).astype(np.float64)
    best = np.argsort(-x, kind="stable")[: keep - (n - age)]
    return sorted(best.tolist()) + list(range(age, n))


def log_softmax(z):
    """Row-wise in 64 bits: minus the largest first, so that a row near the type's lowest value keeps its digits; a row
    of -inf alone stays -inf."""
    top = z.amax(1, keepdim=True)
    d = z - torch.where(top == -math.inf, torch.zeros_like(top), top)
    total = torch.exp(d).sum(1, keepdim=True)
    return torch.where(total == 0, torch.full_like(z, -math.inf), d - torch.log(total)), (top + torch.log(total))[:, 0]


def score(x, scale, tokens, top):
    """lse, logp, entropy, top tokens and their logp of [rows, vocab] values, in 64 bits (the ranking by scale x rounded
    to fp32, which is what is compared)."""
    x32 = (x.float() * scale).float()
    lp, lse = log_softmax(x.double() * scale)
    p = torch.exp(lp)
    ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    logp = torch.where(inside, lp.gather(1, tokens.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0], torch.zeros_like(lse))
    ranked = torch.where(torch.isnan(x32), torch.full_like(x32, -math.inf), x32)
    order = torch.sort(ranked, dim=1, descending=True, stable=True).indices[:, :top]
    return lse, logp, ent, order, lp.gather(1, order)


def score_grad(x, scale, tokens, dlogp, dent):
    lp, lse = log_softmax(x.double() * scale)
    p = torch.exp(lp)
    plp = torch.where(p == 0, torch.zeros_like(p), p * lp)
    ent = -plp.sum(1, keepdim=True)
    inside = ((tokens >= 0) & (tokens < x.shape[1]) & (lse != -math.inf))[:, None]
    g = torch.where(inside, dlogp.double()[:, None], torch.zeros_like(ent))
    hit = torch.zeros_like(lp).scatter_(1, tokens.long().clamp(0, x.shape[1] - 1)[:, None], 1.0)
    return scale * (g * (hit - p) - dent.double()[:, None] * (plp + p * ent))
