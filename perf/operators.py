"""Measured cases of the token-serving operators: the paged key-value cache (append, attention of one new token,
eviction by accumulated attention weight) and the scoring of given tokens (log probabilities, entropy, top
alternatives, and their gradient).

Every case is a dict of plain values. ``prepare`` makes its inputs on the GPU from a seed, ``run`` is one pass over
them: through the library where ``own`` is true, else in plain torch operations in 32 bits, rounded once at the end.
``exact`` gives the same outputs from the operators' definitions in 64 bits. Lengths are spread evenly between
``shortest`` and ``longest`` and dealt to the sequences by the seed, so the work of a case does not depend on it.
"""
import functools
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_BYTES = 1.0e9  # of a drawn case; the largest listed ones move a little more


def listed():
    return [
        # A chat's next token: one sequence, a few hundred tokens of context. All latency.
        dict(name="attend one", op="attend", batch=1, heads=32, kv_heads=8, dim=128, page=16, shortest=417, longest=417,
             window=0, weights=False, type="bf16", heads_first=False),
        # A served batch in the middle of its answers, lengths of every age, grouped heads.
        dict(name="attend batch", op="attend", batch=64, heads=32, kv_heads=8, dim=128, page=64, shortest=1,
             longest=4096, window=0, weights=False, type="bf16", heads_first=True),
        # Two long documents: few rows, so the work has to be split along the cache.
        dict(name="attend long", op="attend", batch=2, heads=64, kv_heads=8, dim=128, page=32, shortest=100_003,
             longest=131_072, window=0, weights=False, type="f16", heads_first=False),
        # A cache that is kept small by eviction: every head its own keys, each step adds up what its keys received.
        dict(name="attend weighted", op="attend", batch=24, heads=16, kv_heads=16, dim=64, page=20, shortest=300,
             longest=2050, window=0, weights=True, type="bf16", heads_first=True),
        # The new token of every sequence of a batch enters the cache.
        dict(name="append token", op="append", batch=64, kv_heads=8, dim=128, page=64, tokens=1, fewest=1,
             shortest=0, longest=4096, type="bf16", heads_first=True),
        # Prompts of several lengths enter it.
        dict(name="append prompts", op="append", batch=6, kv_heads=8, dim=128, page=16, tokens=4096, fewest=1000,
             shortest=0, longest=700, type="f16", heads_first=False),
        # One sequence has outgrown its budget by a few tokens.
        dict(name="evict one", op="evict", batch=1, kv_heads=8, dim=128, page=32, shortest=1051, longest=1051,
             keep=1024, recent=256, type="bf16", heads_first=False),
        # A batch of long prompts is cut to a budget; the short ones among them are taken whole.
        dict(name="evict batch", op="evict", batch=16, kv_heads=8, dim=128, page=64, shortest=3000, longest=16_000,
             keep=4096, recent=512, type="bf16", heads_first=True),
        # What a server reports of the tokens it has just chosen.
        dict(name="score step", op="score", rows=8, vocab=131_072, top=20, entropy=True, scale=1.0, type="bf16", masked=0.0),
        # The answers of a batch are scored again; a vocabulary of odd width, sampled at a temperature.
        dict(name="score answers", op="score", rows=4096, vocab=50_257, top=5, entropy=True, scale=1.25, type="bf16", masked=0.01),
        # The gradient of a small update in 32 bits.
        dict(name="score grad small", op="grad", rows=48, vocab=32_000, entropy=False, scale=1.0, type="f32", masked=0.0),
        # The gradient of a policy's update over a large vocabulary, with its entropy.
        dict(name="score grad", op="grad", rows=2048, vocab=131_072, entropy=True, scale=1.0, type="bf16", masked=0.0),
    ]


def draw(rng):
    """One more case: an operator, then sizes spread over the logarithm of their range until the case is not too large."""
    def size(low, high):
        return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))

    op = rng.choice(("attend", "attend", "append", "evict", "score", "grad"))
    while True:
        if op in ("score", "grad"):
            case = dict(op=op, rows=size(1, 4096), vocab=size(1000, 160_000), entropy=rng.random() < 0.6,
                        scale=rng.choice((1.0, 0.7, 1.25)), type=rng.choice(("bf16", "f16", "f32")), masked=rng.choice((0.0, 0.02)))
            if op == "score":
                case["top"] = rng.choice((0, 1, 5, 20, 32))
        else:
            kv_heads = rng.choice((1, 2, 4, 8, 8, 16))
            case = dict(op=op, batch=size(1, 128), kv_heads=kv_heads, dim=rng.choice((64, 128, 128, 256)),
                        page=rng.choice((1, 8, 16, 16, 20, 32, 64, 128)), type=rng.choice(("bf16", "f16")), heads_first=rng.random() < 0.5)
            if op == "append":
                tokens = rng.choice((1, 1, size(2, 4096)))
                longest = size(1, 8192)
                case.update(tokens=tokens, fewest=rng.randint(1, tokens), shortest=rng.randint(0, longest), longest=longest)
            else:
                longest = size(1 if op == "attend" else 64, 100_000)
                case.update(shortest=rng.choice((longest, rng.randint(0, longest))), longest=longest)
            if op == "attend":
                case.update(heads=kv_heads * rng.choice((1, 2, 4, 7, 8, 16)), window=rng.choice((0, 0, size(1, 8192))),
                            weights=rng.random() < 0.4)
            if op == "evict":
                keep = max(1, int(longest * rng.uniform(0.1, 1.0)))
                case.update(keep=keep, recent=rng.randint(0, keep))
        if 2e3 < held(case) < 4e9 and work(case)["bytes"] <= MOST_BYTES:
            return case


def lengths(case):
    """The sequences' lengths, in rising order."""
    b = case["batch"]
    return [case["shortest"] + (case["longest"] - case["shortest"]) * i // max(1, b - 1) for i in range(b)]


def counts(case):
    """How many new tokens the sequences bring, in rising order."""
    b = case["batch"]
    return [case["fewest"] + (case["tokens"] - case["fewest"]) * i // max(1, b - 1) for i in range(b)]


def held(case):
    """Bytes of the 32-bit copies that the plain form makes of a case's largest tensors, about."""
    if "vocab" in case:
        return 4.0 * case["rows"] * case["vocab"]
    return 8.0 * case["batch"] * case["kv_heads"] * case["dim"] * (case["longest"] + case.get("tokens", 0))


def work(case):
    """What a pass cannot do without: every input read once, every output written once, the operations of the sums."""
    if case["op"] in ("score", "grad"):
        rows, cells, size = case["rows"], case["rows"] * case["vocab"], torch.finfo(TYPES[case["type"]]).bits // 8
        if case["op"] == "score":
            return {"bytes": cells * size + rows * (12 + 4 * case["entropy"] + 8 * case["top"]), "flops": cells * (6 if case["entropy"] else 4)}
        return {"bytes": 2 * cells * size + rows * (12 + 8 * case["entropy"]), "flops": cells * (8 if case["entropy"] else 4)}
    row = 2 * 2 * case["kv_heads"] * case["dim"]  # K and V of one token
    if case["op"] == "append":
        return {"bytes": 2 * row * sum(counts(case)) + 12 * case["batch"], "flops": 0}
    lens = lengths(case)
    if case["op"] == "evict":
        slots, kept = sum(lens), sum(min(n, case["keep"]) for n in lens)
        return {"bytes": 2 * row * kept + case["kv_heads"] * (4 * slots + 8 * kept), "flops": case["kv_heads"] * slots}
    seen = sum(min(n, case["window"] or n) for n in lens)
    both = 2 * 2 * case["batch"] * case["heads"] * case["dim"]
    return {"bytes": row * seen + both + 4 * case["batch"] * case["heads"] + (8 * seen * case["kv_heads"] if case["weights"] else 0),
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ inputs

@functools.cache
def library():
    """The library's module and the handle that a program keeps."""
    from grxcp_b200 import dnn
    return dnn, dnn.Handle()


def paged(case, gen, tokens, fill):
    """Pools of pages [pages, page, kv_heads, dim] for sequences of so many tokens, and their table: pages lie in no order, entries that no
    token needs are -1, and two pages belong to nobody."""
    page, dev = case["page"], "cuda"
    need = (tokens + page - 1) // page
    width, total = max(1, int(need.max())), int(need.sum())
    shape = (total + 2, case["kv_heads"], page, case["dim"]) if case["heads_first"] else (total + 2, page, case["kv_heads"], case["dim"])
    pools = [torch.randn(shape, device=dev, dtype=TYPES[case["type"]], generator=gen) if fill else
             torch.zeros(shape, device=dev, dtype=TYPES[case["type"]]) for _ in range(2)]
    if case["heads_first"]:
        pools = [p.transpose(1, 2) for p in pools]
    at = (torch.cumsum(need, 0) - need)[:, None] + torch.arange(width, device=dev)
    order = torch.randperm(total + 2, device=dev, generator=gen)
    table = torch.where(torch.arange(width, device=dev) < need[:, None], order[at.clamp(max=total + 1)], -1)
    return pools[0], pools[1], table.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind = "cuda", TYPES[case["type"]]
    state = {"case": case}

    def normal(*shape, kind=torch.float32):
        return torch.randn(*shape, device=dev, dtype=kind, generator=gen)

    if case["op"] in ("score", "grad"):
        rows, vocab = case["rows"], case["vocab"]
        # A model's logits: a spread of about 2.5, a few tokens that stand out, and some that a grammar forbids.
        logits = torch.empty(rows, vocab, device=dev, dtype=kind)
        logits.normal_(0.0, 2.5, generator=gen)
        tokens = torch.randint(vocab, (rows,), device=dev, generator=gen)
        likely = torch.randint(vocab, (rows, 4), device=dev, generator=gen)
        logits.scatter_(1, likely, (12.0 + 2.0 * normal(rows, 4)).to(kind))
        tokens = torch.where(torch.rand(rows, device=dev, generator=gen) < 0.7, likely[:, 0], tokens)
        if case["masked"]:
            forbidden = torch.randint(vocab, (rows, max(1, int(case["masked"] * vocab))), device=dev, generator=gen)
            forbidden = torch.where(forbidden == tokens[:, None], likely[:, 1:2], forbidden)
            logits.scatter_(1, forbidden, float("-inf"))
            logits.scatter_(1, tokens[:, None], 11.0)
        state.update(logits=logits, tokens=tokens.to(torch.int32))
        f = dict(device=dev, dtype=torch.float32)
        if case["op"] == "score":
            state.update(logp=torch.empty(rows, **f), lse=torch.empty(rows, **f), entropy=torch.empty(rows, **f) if case["entropy"] else None,
                         top_tokens=torch.empty(rows, case["top"], device=dev, dtype=torch.int32) if case["top"] else None,
                         top_logp=torch.empty(rows, case["top"], **f) if case["top"] else None)
        else:
            lse, entropy = statistics(logits, case["scale"])
            state.update(lse=lse, entropy=entropy if case["entropy"] else None, dlogp=normal(rows),
                         dentropy=0.01 * normal(rows) if case["entropy"] else None, dlogits=torch.empty_like(logits))
        return state
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["dim"]
    deal = torch.randperm(batch, device=dev, generator=gen)
    lens = torch.tensor(lengths(case), device=dev)[deal]
    new = torch.tensor(counts(case), device=dev)[deal] if case["op"] == "append" else 0
    k, v, table = paged(case, gen, lens + new, True)
    state.update(k=k, v=v, table=table, lens=lens.to(torch.int32))
    if case["op"] == "append":
        state.update(new_k=normal(batch, case["tokens"], kv_heads, dim, kind=kind).transpose(1, 2),
                     new_v=normal(batch, case["tokens"], kv_heads, dim, kind=kind).transpose(1, 2),
                     counts=new.to(torch.int32), lens_out=torch.empty(batch, device=dev, dtype=torch.int32))
    elif case["op"] == "attend":
        state.update(q=(2.0 * normal(batch, case["heads"], 1, dim)).to(kind), o=torch.empty(batch, case["heads"], 1, dim, device=dev, dtype=kind),
                     lse=torch.empty(batch, case["heads"], device=dev), scale=dim ** -0.5, weights=None)
        if case["weights"]:
            state["weights"] = normal(batch, kv_heads, table.shape[1] * case["page"]).square()
    else:
        slots = torch.arange(table.shape[1] * case["page"], device=dev)
        weights = torch.exp(2.0 * normal(batch, kv_heads, slots.numel()))  # a few keys receive most; some nothing, and tie
        weights = torch.where(torch.rand(weights.shape, device=dev, generator=gen) < 0.1, 0.0, weights)
        k_out, v_out, table_out = paged(case, gen, lens.clamp(max=case["keep"]).clamp(min=1), False)
        width = -(-case["keep"] // case["page"])  # room for `keep` in every table row; pages that no sequence needs are not there
        table_out = torch.nn.functional.pad(table_out, (0, max(0, width - table_out.shape[1])), value=-1)
        state.update(weights=torch.where(slots < lens[:, None, None], weights, 0.0), k_out=k_out, v_out=v_out, table_out=table_out,
                     lens_out=torch.empty(batch, device=dev, dtype=torch.int32),
                     weights_out=torch.empty(batch, kv_heads, table_out.shape[1] * case["page"], device=dev),
                     indices=torch.empty(batch, kv_heads, case["keep"], device=dev, dtype=torch.int32))
    if own:
        dnn, _ = library()
        state["cache"] = dnn.PagedCache(state["k"], state["v"], state["table"])
        if case["op"] == "evict":
            state["cache_out"] = dnn.PagedCache(state["k_out"], state["v_out"], state["table_out"])
    return state


# ------------------------------------------------------------------ passes

def run(state):
    op = state["case"]["op"]
    return (OWN if own else PLAIN)[op](state)


def own_attend(s):
    dnn, h = library()
    dnn.check(h.paged_attention(s["cache"], s["lens"], s["q"], s["o"], s["scale"], s["case"]["window"], s["lse"], s["weights"]))
    return {"o": s["o"], "lse": s["lse"], "weights": s["weights"]}


def own_append(s):
    dnn, h = library()
    dnn.check(h.kv_append(s["cache"], s["lens"], s["new_k"], s["new_v"], s["counts"], s["lens_out"]))
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"]}


def own_evict(s):
    dnn, h = library()
    dnn.check(h.kv_evict(s["cache"], s["lens"], s["weights"], s["case"]["keep"], s["case"]["recent"], s["cache_out"], s["lens_out"],
                         s["weights_out"], s["indices"]))
    return {"k": s["k_out"], "v": s["v_out"], "lens": s["lens_out"], "weights": s["weights_out"], "indices": s["indices"]}


def own_score(s):
    dnn, h = library()
    dnn.check(h.token_logprobs(s["logits"], s["tokens"], s["logp"], s["case"]["scale"], s["entropy"], s["lse"], s["top_tokens"], s["top_logp"]))
    return {n: s[n] for n in ("logp", "lse", "entropy", "top_tokens", "top_logp")}


def own_grad(s):
    dnn, h = library()
    dnn.check(h.token_logprobs_backward(s["logits"], s["tokens"], s["lse"], s["dlogp"], s["dlogits"], s["case"]["scale"], s["entropy"],
                                        s["dentropy"]))
    return {"dlogits": s["dlogits"]}


OWN = {"attend": own_attend, "append": own_append, "evict": own_evict, "score": own_score, "grad": own_grad}


def gathered(pages, table):
    """The tokens of every sequence in order, [batch, kv_heads, tokens, dim]."""
    return pages[table.long().clamp(min=0)].flatten(1, 2).transpose(1, 2)


def plain_attend(s):
    case = s["case"]
    k, v = (gathered(s[n], s["table"]).float() for n in ("k", "v"))
    b, h, n, d = k.shape
    q = s["q"].float().reshape(b, h, -1, d)
    slot = torch.arange(n, device=q.device)
    lens = s["lens"].long()[:, None]
    seen = slot < lens
    if case["window"]:
        seen &= slot >= lens - case["window"]
    seen = seen[:, None, None, :]
    scores = torch.where(seen, torch.matmul(q, k.transpose(2, 3)) * s["scale"], -math.inf)
    top = scores.amax(3, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    share = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(share, torch.where(seen.transpose(2, 3), v, 0.0))
    s["o"].copy_(o.reshape(s["o"].shape))
    s["lse"].copy_((top + torch.log(total)).reshape(s["lse"].shape))
    if s["weights"] is not None:
        s["weights"] += share.sum(2)
    return {"o": s["o"], "lse": s["lse"], "weights": s["weights"]}


def plain_append(s):
    page = s["case"]["page"]
    t = torch.arange(s["case"]["tokens"], device=s["k"].device)
    b, i = torch.nonzero(t < s["counts"][:, None], as_tuple=True)
    at = s["lens"][b].long() + i
    where = s["table"][b, at // page].long()
    s["k"][where, at % page] = s["new_k"][b, :, i]
    s["v"][where, at % page] = s["new_v"][b, :, i]
    torch.add(s["lens"], s["counts"], out=s["lens_out"])
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"]}


def plain_evict(s):
    keep, recent, page = s["case"]["keep"], s["case"]["recent"], s["case"]["page"]
    w = s["weights"]
    slot = torch.arange(w.shape[2], device=w.device)
    lens = s["lens"].long()[:, None, None]
    count = lens.clamp(max=keep)
    rank = torch.where(slot >= lens - recent, math.inf, w)
    rank = torch.where(slot >= lens, -math.inf, rank)
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    best = torch.nn.functional.pad(best, (0, keep - best.shape[2]), value=w.shape[2])
    i = torch.arange(keep, device=w.device)
    best = torch.sort(torch.where(i < count, best, w.shape[2]), dim=2).values
    s["indices"].copy_(torch.where(i < count, best, -1))
    s["lens_out"].copy_(count.flatten())
    b, h, j = torch.nonzero(i < count.expand(-1, w.shape[1], -1), as_tuple=True)
    src = best[b, h, j]
    for_out = s["table_out"][b, j // page].long()
    from_in = s["table"][b, src // page].long()
    s["k_out"][for_out, j % page, h] = s["k"][from_in, src % page, h]
    s["v_out"][for_out, j % page, h] = s["v"][from_in, src % page, h]
    s["weights_out"].zero_()
    s["weights_out"][b, h, j] = w[b, h, src]
    return {"k": s["k_out"], "v": s["v_out"], "lens": s["lens_out"], "weights": s["weights_out"], "indices": s["indices"]}


def statistics(logits, scale):
    """log of the sum of the exponentials, and the entropy, of each row in 32 bits."""
    x = logits.float() * scale
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    mean = torch.where(e > 0, e * (x - top), 0.0).sum(1, keepdim=True) / total
    return (top + torch.log(total)).flatten(), (torch.log(total) - mean).flatten()


def plain_score(s):
    case = s["case"]
    lse, entropy = statistics(s["logits"], case["scale"])
    x = s["logits"].float() * case["scale"]
    s["lse"].copy_(lse)
    s["logp"].copy_(x.gather(1, s["tokens"].long()[:, None]).flatten() - lse)
    if case["entropy"]:
        s["entropy"].copy_(entropy)
    if case["top"]:
        values, places = torch.sort(x, dim=1, descending=True, stable=True)  # equal ones stay in the order of their tokens
        s["top_tokens"].copy_(places[:, : case["top"]])
        s["top_logp"].copy_(values[:, : case["top"]] - lse[:, None])
    return {n: s[n] for n in ("logp", "lse", "entropy", "top_tokens", "top_logp")}


def plain_grad(s):
    scale, lse = s["case"]["scale"], s["lse"][:, None]
    x = s["logits"].float() * scale
    p = torch.exp(x - lse)
    g = -s["dlogp"][:, None] * p
    if s["dentropy"] is not None:
        g -= s["dentropy"][:, None] * torch.where(p > 0, p * (x - lse + s["entropy"][:, None]), 0.0)
    g.scatter_add_(1, s["tokens"].long()[:, None], s["dlogp"][:, None])
    s["dlogits"].copy_(g * scale)
    return {"dlogits": s["dlogits"]}


PLAIN = {"attend": plain_attend, "append": plain_append, "evict": plain_evict, "score": plain_score, "grad": plain_grad}


# ------------------------------------------------------------------ definitions in 64 bits

def exact(case, seed):
    return EXACT[case["op"]](case, prepare(case, seed))


def of_one(pages, table, n, page):
    """The first n tokens of one sequence, [n, kv_heads, dim]."""
    return torch.cat([pages[int(p)] for p in table[: -(-n // page)].tolist()])[:n] if n else pages[0][:0]


def exact_attend(case, s):
    group, out = case["heads"] // case["kv_heads"], {"o": [], "lse": []}
    weights = None if s["weights"] is None else s["weights"].double()
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        k, v = (of_one(s[x], s["table"][b], n, case["page"])[first:].double() for x in ("k", "v"))
        if n == first:
            out["o"].append(torch.zeros_like(s["o"][b], dtype=torch.float64))
            out["lse"].append(torch.full_like(s["lse"][b], -math.inf, dtype=torch.float64))
            continue
        q = s["q"][b, :, 0].double().unflatten(0, (-1, group))
        logits = torch.einsum("hgd,nhd->hgn", q, k) * s["scale"]
        out["o"].append(torch.einsum("hgn,nhd->hgd", logits.softmax(2), v).reshape(-1, 1, case["dim"]))
        out["lse"].append(logits.logsumexp(2).flatten())
        if weights is not None:
            weights[b, :, first:n] += logits.softmax(2).sum(1)
    return {"o": torch.stack(out["o"]), "lse": torch.stack(out["lse"]), "weights": weights}


def exact_append(case, s):
    k, v, page = s["k"].double(), s["v"].double(), case["page"]
    for b, (n, new) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
        row = s["table"][b].tolist()
        t = 0
        while t < new:  # page by page
            at = (n + t) % page
            m = min(page - at, new - t)
            k[row[(n + t) // page], at:at + m] = s["new_k"][b, :, t:t + m].transpose(0, 1).double()
            v[row[(n + t) // page], at:at + m] = s["new_v"][b, :, t:t + m].transpose(0, 1).double()
            t += m
    return {"k": k, "v": v, "lens": s["lens"] + s["counts"]}


def exact_evict(case, s):
    keep, page = case["keep"], case["page"]
    k, v = s["k_out"].double(), s["v_out"].double()
    weights, indices = torch.zeros_like(s["weights_out"], dtype=torch.float64), torch.full_like(s["indices"], -1)
    for b, n in enumerate(s["lens"].tolist()):
        old = [of_one(s[x], s["table"][b], n, page).double() for x in ("k", "v")]
        m = min(n, keep)
        at = torch.arange(m, device=k.device)
        pages = s["table_out"][b].long()[at // page]
        for h in range(case["kv_heads"]):
            w = s["weights"][b, h, :n].double().cpu().numpy()
            age = n - min(n, case["recent"])
            kept = list(range(n)) if n <= keep else sorted((-w[:age]).argsort(kind="stable")[: keep - (n - age)].tolist()) + list(range(age, n))
            kept = torch.tensor(kept, device=k.device, dtype=torch.long)
            indices[b, h, :m] = kept.int()
            weights[b, h, :m] = s["weights"][b, h][kept].double()
            k[pages, at % page, h] = old[0][kept, h]
            v[pages, at % page, h] = old[1][kept, h]
    return {"k": k, "v": v, "lens": s["lens"].clamp(max=keep), "weights": weights, "indices": indices}


def exact_score(case, s):
    out = {"logp": [], "lse": [], "entropy": [], "top_logp": []}
    for rows, tokens in zip(s["logits"].split(64), s["tokens"].long().split(64)):
        logp = torch.log_softmax(rows.double() * case["scale"], 1)
        out["logp"].append(logp.gather(1, tokens[:, None])[:, 0])
        out["lse"].append(torch.logsumexp(rows.double() * case["scale"], 1))
        out["entropy"].append(-torch.xlogy(logp.exp(), logp.exp()).sum(1))
        out["top_logp"].append(logp.topk(case["top"], 1).values)
    out = {n: torch.cat(x) for n, x in out.items()}
    return {"logp": out["logp"], "lse": out["lse"], "entropy": out["entropy"] if case["entropy"] else None,
            "top_tokens": None, "top_logp": out["top_logp"] if case["top"] else None}


def exact_grad(case, s):
    """The derivative along each logit of dlogp * logp + dentropy * entropy, at the statistics that the pass is given."""
    got = torch.empty_like(s["logits"], dtype=torch.float64)
    zero = torch.zeros((), device=got.device, dtype=torch.float64)
    for r in range(0, case["rows"], 64):
        part = slice(r, r + 64)
        logp = s["logits"][part].double() * case["scale"] - s["lse"][part, None].double()
        hit = torch.zeros_like(logp).scatter_(1, s["tokens"][part, None].long(), 1.0)
        d = s["dlogp"][part, None].double() * (hit - logp.exp())
        if case["entropy"]:
            d = d - s["dentropy"][part, None].double() * (torch.where(logp.exp() > 0, logp, zero) + s["entropy"][part, None].double()) * logp.exp()
        got[part] = d * case["scale"]
    return {"dlogits": got}


EXACT = {"attend": exact_attend, "append": exact_append, "evict": exact_evict, "score": exact_score, "grad": exact_grad}
