"""The serving operators over a paged key-value cache, and the log probabilities of a step's tokens: cases to measure.

A case's ``op`` says which operator it is:

* ``append``    rotary embedding of the tokens of a step (or of prompts) and their keys and values written into pages;
* ``attend``    attention of one new token per sequence over its pages, optionally adding each cached position's
  attention weight (summed over the query heads that share a key-value head) to an accumulator;
* ``evict``     the positions of highest accumulated weight, and the most recent ones, kept and copied in order into
  new pages;
* ``logprobs``  log probabilities of given tokens with the entropy and the top alternatives of each row of logits.

``run`` computes them in plain torch, or, where ``own`` is true, by the calls a user of the package makes.  The
cache is ``[pages, kv_heads, page, head_dim]`` (``layout`` "heads") or the same view of ``[pages, page, kv_heads,
head_dim]`` memory (``layout`` "tokens"); ``table[b, i]`` is the page that holds positions ``i * page`` onwards of
sequence ``b``.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    cache = {"heads": 32, "kv_heads": 8, "dim": 64, "layout": "heads", "dtype": "bf16"}  # the Llama-3.2-1B-shaped model's
    return [
        # the first steps of a chat with one user: latency alone counts
        {"name": "attend, one short sequence", "op": "attend", "seqs": 1, "longest": 137, "page": 16, "weights": False, **cache},
        # a server's ordinary batch: sequences of all ages, one of them empty, none of them a whole number of pages
        {"name": "attend, ragged batch", "op": "attend", "seqs": 32, "longest": 2047, "page": 64, "weights": False, **cache},
        # few long documents: the cache's length is the only axis to split over
        {"name": "attend, four long sequences", "op": "attend", "seqs": 4, "longest": 131072, "page": 128, "weights": False,
         **cache, "dtype": "fp16"},
        # a wider head and a larger group of query heads, tokens' heads next to each other in memory
        {"name": "attend, wide heads", "op": "attend", "seqs": 24, "longest": 8191, "page": 32, "weights": False,
         "heads": 64, "kv_heads": 8, "dim": 128, "layout": "tokens", "dtype": "bf16"},
        # serving under a cache budget: each step also adds up what every position was attended with
        {"name": "attend, weights accumulated", "op": "attend", "seqs": 8, "longest": 16384, "page": 32, "weights": True, **cache},
        # one decode step's tokens: a launch that has to be short
        {"name": "append, decode step", "op": "append", "tokens": 8, "seqs": 8, "longest": 1024, "page": 16, **cache},
        # the prompts of a batch, packed one behind the other
        {"name": "append, prompts", "op": "append", "tokens": 16381, "seqs": 9, "longest": 4096, "page": 64, **cache},
        # one conversation halved when it reaches its budget
        {"name": "evict, one sequence", "op": "evict", "seqs": 1, "longest": 2048, "budget": 1024, "recent": 128, "page": 16, **cache},
        # a batch of long contexts cut to a quarter
        {"name": "evict, long batch", "op": "evict", "seqs": 16, "longest": 32768, "budget": 8192, "recent": 1000, "page": 64, **cache},
        # the answer of one decode step with its alternatives
        {"name": "logprobs, one step", "op": "logprobs", "rows": 1, "vocab": 128256, "top": 5, "masked": 0.0, "dtype": "bf16"},
        # a batch's step under a grammar that leaves few tokens, an odd vocabulary, 32-bit logits
        {"name": "logprobs, constrained batch", "op": "logprobs", "rows": 61, "vocab": 100003, "top": 20, "masked": 0.9, "dtype": "fp32"},
        # scoring a text: one sequence of the model's perplexity check
        {"name": "logprobs, scored text", "op": "logprobs", "rows": 2048, "vocab": 128256, "top": 0, "masked": 0.0, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, int(round(lo * (hi / lo) ** rng.random())))

    op = rng.choice(["attend", "attend", "append", "evict", "logprobs"])
    if op == "logprobs":
        dtype, vocab = rng.choice(["bf16", "fp16", "fp32"]), log(1000, 200000)
        return {"op": op, "rows": min(log(1, 2048), (1 << 28) // vocab), "vocab": vocab, "top": rng.choice([0, 1, rng.randint(2, 20)]),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.99]), "dtype": dtype}
    kv_heads, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 64, 128])
    case = {"op": op, "heads": kv_heads * rng.choice([1, 2, 4, 4, 7, 8]), "kv_heads": kv_heads, "dim": dim,
            "layout": rng.choice(["heads", "heads", "tokens"]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "page": rng.choice([8, 16, 24, 32, 64, 128, 256])}
    row = kv_heads * dim * 4  # bytes of a position's keys and values
    if op == "append":
        case["seqs"] = log(1, 64)
        case["longest"] = log(16, 8192)
        case["tokens"] = min(log(case["seqs"], 16384), case["seqs"] * (case["longest"] // 2))
        case["tokens"] = max(case["tokens"], case["seqs"])
        return case
    case["seqs"] = log(1, 128)
    case["longest"] = min(log(1 if op == "attend" else 64, 131072), max(64, (1 << 29) // (row * case["seqs"])))
    if op == "attend":
        case["weights"] = rng.random() < 0.35
    else:
        case["budget"] = rng.randint(1, max(1, case["longest"] // 2))
        case["recent"] = rng.randint(0, case["budget"])
    return case


# ------------------------------------------------------------------ what a program has in hand


def _lens(case):
    """Lengths of the sequences: the longest, and others spread below it; one in seven or so of a batch is empty or one long."""
    r = random.Random("%s %s %s" % (case["op"], case["seqs"], case["longest"]))
    n = [max(1, int(case["longest"] * (0.25 + 0.75 * r.random()))) for _ in range(case["seqs"])]
    n[0] = case["longest"]
    if case["op"] == "attend":
        for b in range(7, len(n), 9):
            n[b] = r.choice([0, 1])
    return n


def _new_tokens(case):
    """How many of the step's tokens belong to each sequence."""
    base, more = divmod(case["tokens"], case["seqs"])
    return [base + (b < more) for b in range(case["seqs"])]


def _pages(n, case):
    return -(-n // case["page"])


def _pool(case, pages, gen, fill):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["layout"] == "tokens":
        shape = (pages, case["page"], case["kv_heads"], case["dim"])
    x = torch.empty(shape, device="cuda", dtype=DTYPES[case["dtype"]])
    if fill is None:
        x.normal_(generator=gen)
    else:
        x.fill_(fill)
    return x.transpose(1, 2) if case["layout"] == "tokens" else x


def _int32(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.empty(rows, vocab, device="cuda", dtype=dtype).normal_(std=3.0, generator=gen)
        targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        if case["masked"] > 0:  # the tokens a grammar rules out; the given ones are among the others
            for r in range(rows):
                out = torch.rand(vocab, device="cuda", generator=gen) < case["masked"]
                out[targets[r]] = False
                logits[r].masked_fill_(out, -math.inf)
        if rows > 4:  # padding
            targets[3] = -1
        return {"case": case, "logits": logits, "targets": targets}
    B, nq, nkv, dim, page = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lens(case)
    if case["op"] == "append":
        new = _new_tokens(case)
        had = [min(n, case["longest"] - k) if case["longest"] > k else 0 for n, k in zip(lens, new)]
        width = max(_pages(h + k, case) for h, k in zip(had, new))
        pages = B * width
        slots = [had[b] + i for b in range(B) for i in range(new[b])]
        seqs = [b for b in range(B) for _ in range(new[b])]
        most = max(slots) + 1 + 37  # positions run ahead of the slots once something was evicted
        inv = 500000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        ang = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * torch.cat([inv, inv])[None]
        # the projection writes into a wider buffer: rows are not packed
        qkv = torch.empty(case["tokens"], (nq + 2 * nkv) * dim + 64, device="cuda", dtype=dtype).normal_(generator=gen)
        return {"case": case, "qkv": qkv[:, : (nq + 2 * nkv) * dim], "cos": ang.cos().to(dtype), "sin": ang.sin().to(dtype),
                "positions": _int32([s + 37 for s in slots]), "slots": _int32(slots), "seqs": _int32(seqs),
                "table": torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).view(B, width),
                "k": _pool(case, pages, gen, 0.0), "v": _pool(case, pages, gen, 0.0)}
    width = max(1, _pages(max(lens), case))
    used = sum(_pages(n, case) for n in lens)
    order = torch.randperm(used, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros(B, width, device="cuda", dtype=torch.int32)  # entries behind a sequence's last page name page 0
    at = 0
    for b, n in enumerate(lens):
        table[b, : _pages(n, case)] = order[at: at + _pages(n, case)]
        at += _pages(n, case)
    state = {"case": case, "table": table, "lens": _int32(lens)}
    if case["op"] == "attend":
        state["k"], state["v"] = _pool(case, max(1, used), gen, None), _pool(case, max(1, used), gen, None)
        for b, n in enumerate(lens):  # what lies behind a sequence's end in its last page is whatever was there before
            if n % page:
                state["k"][table[b, n // page], :, n % page:] = math.nan
                state["v"][table[b, n // page], :, n % page:] = math.nan
        state["q"] = (torch.empty(B, nq, dim, device="cuda").normal_(std=1.5, generator=gen)).to(dtype)
        if case["weights"]:
            state["weights"] = torch.rand(B, nkv, width * page, device="cuda", generator=gen)
    else:
        kept = [min(n, case["budget"]) for n in lens]
        new_width = _pages(case["budget"], case)
        pages = used + B * new_width
        state["k"], state["v"] = _pool(case, pages, gen, None), _pool(case, pages, gen, None)
        state["new_table"] = (used + torch.randperm(B * new_width, device="cuda", generator=gen).to(torch.int32)).view(B, new_width)
        # accumulated weight: a heavy tail, and positions that were never looked at
        w = torch.rand(B, nkv, width * page, device="cuda", generator=gen)
        w = (0.02 / (w + 1e-3)) * torch.rand(w.shape, device="cuda", generator=gen)
        state["weights"] = torch.where(torch.rand(w.shape, device="cuda", generator=gen) < 0.1, 0.0, w)
        assert max(kept) > 0
    return state


# ------------------------------------------------------------------ one pass


def _ops():
    at = os.path.join(os.getcwd(), "itmo-final-project_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import int4_b200

    return int4_b200


def _own(s):
    ops, case = _ops(), s["case"]
    if case["op"] == "logprobs":
        lp, entropy, top_lp, top_ids = ops.token_logprobs(s["logits"], s["targets"], top=case["top"])
        return (lp, entropy, top_lp, top_ids) if case["top"] else (lp, entropy)
    if case["op"] == "append":
        q = ops.paged_kv_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["table"], s["k"], s["v"], seqs=s["seqs"])
        return q, s["k"], s["v"]
    if case["op"] == "attend":
        out = ops.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], weights=s.get("weights"))
        return (out, s["weights"]) if case["weights"] else (out,)
    lens, kept, weights = ops.paged_evict(s["weights"], s["lens"], s["table"], s["k"], s["v"], s["new_table"], case["budget"],
                                          recent=case["recent"])
    return lens, kept, weights, s["k"], s["v"]


def run(s):
    if own:
        return _own(s)
    return {"logprobs": _plain_logprobs, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[s["case"]["op"]](s)


def _plain_logprobs(s):
    top, targets = s["case"]["top"], s["targets"]
    z = s["logits"].float()
    best = z.max(-1, keepdim=True).values
    d = z - best
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    entropy = (lse - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total).squeeze(-1)
    got = (torch.gather(d, 1, targets.clamp_min(0)[:, None]) - lse).squeeze(-1)
    got = torch.where(targets < 0, 0.0, got)
    if not top:
        return got, entropy
    bits = z.view(torch.int32).to(torch.int64)
    bits = torch.where(bits < 0, -2147483648 - bits, bits)  # in the order of the values; -0 as +0
    key = bits * (1 << 24) + (z.shape[-1] - 1 - torch.arange(z.shape[-1], device=z.device))  # ties: the lowest index
    ids = torch.topk(key, top, dim=-1).indices
    return got, entropy, torch.gather(d, 1, ids) - lse, ids


def _plain_append(s):
    case, dtype = s["case"], s["k"].dtype
    nq, nkv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    x = s["qkv"].reshape(case["tokens"], nq + 2 * nkv, dim).float()
    at = s["positions"].long()
    cos, sin = s["cos"].float()[at][:, None], s["sin"].float()[at][:, None]
    t, v = x[:, : nq + nkv], x[:, nq + nkv:]
    t = t * cos + torch.cat([-t[..., dim // 2:], t[..., : dim // 2]], -1) * sin
    slot = s["slots"].long()
    where = s["table"][s["seqs"].long(), slot // page].long()
    s["k"][where, :, slot % page] = t[:, nq:].to(dtype)
    s["v"][where, :, slot % page] = v.to(dtype)
    return t[:, :nq].to(dtype), s["k"], s["v"]


def _plain_attend(s):
    case = s["case"]
    B, nq, nkv, dim = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    k = s["k"][s["table"].long()].transpose(1, 2).reshape(B, nkv, -1, dim)
    v = s["v"][s["table"].long()].transpose(1, 2).reshape(B, nkv, -1, dim)
    here = torch.arange(k.shape[2], device="cuda")[None] < s["lens"][:, None]
    q = s["q"].float().view(B, nkv, nq // nkv, dim)
    logit = (torch.matmul(q, k.float().transpose(-1, -2)) * dim ** -0.5).masked_fill(~here[:, None, None], -math.inf)
    best = logit.max(-1, keepdim=True).values.clamp_min(-3e38)
    p = torch.exp(logit - best)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = torch.where(here[:, None, :, None], v, 0.0).float()
    out = torch.matmul(p, v).view(B, nq, dim).to(s["q"].dtype)
    if not case["weights"]:
        return (out,)
    s["weights"] += p.sum(2)
    return out, s["weights"]


def _plain_evict(s):
    case = s["case"]
    budget, page, nkv = case["budget"], case["page"], case["kv_heads"]
    w, lens = s["weights"], s["lens"].long()
    n = torch.arange(w.shape[-1], device="cuda")[None]
    kept_len = lens.clamp_max(budget)
    # the recent ones rank above everything, positions behind the end below; ties go to the lowest position
    rank = torch.where(n >= lens[:, None], -1.0, torch.where(n >= (lens - case["recent"])[:, None], math.inf, 0.0))[:, None]
    order = torch.sort(torch.where(rank == 0.0, w, rank), dim=-1, descending=True, stable=True).indices
    first = torch.arange(budget, device="cuda")
    some = (first[None] < kept_len[:, None])[:, None]
    if order.shape[-1] < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]))
    idx = torch.where(some, order[..., :budget], w.shape[-1]).sort(-1).values
    src = torch.where(some, idx, 0)
    kept = torch.where(some, idx, -1).to(torch.int32)
    new_w = torch.zeros_like(w)
    m = min(budget, w.shape[-1])
    new_w[..., :m] = torch.where(some, torch.gather(w, -1, src), 0.0)[..., :m]
    from_page = torch.gather(s["table"].long()[:, None].expand(-1, nkv, -1), -1, src // page)
    to_page = s["new_table"].long()[:, None, first // page].expand(-1, nkv, -1)
    head = torch.arange(nkv, device="cuda")[None, :, None].expand_as(src)
    every = some.expand_as(src)
    for c in (s["k"], s["v"]):
        c[to_page[every], head[every], (first % page).expand_as(src)[every]] = c[from_page[every], head[every], (src % page)[every]]
    return kept_len.to(torch.int32), kept, new_w, s["k"], s["v"]


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    nq, nkv, dim, B = case["heads"], case["kv_heads"], case["dim"], case["seqs"]
    if case["op"] == "append":
        T = case["tokens"]
        # read q, k and v and a row of each table, write them; positions, slots, sequences and pages
        return {"bytes": T * (4 * (nq + 2 * nkv) * dim + 4 * dim + 16), "flops": 3 * T * (nq + nkv) * dim}
    total = sum(_lens(case))
    if case["op"] == "attend":
        b = 4 * nkv * dim * total + 4 * B * nq * dim + 4 * (total // case["page"] + 2 * B)
        return {"bytes": b + (8 * nkv * total if case["weights"] else 0), "flops": 4 * nq * dim * total}
    kept = sum(min(n, case["budget"]) for n in _lens(case))
    width = max(_lens(case))
    return {"bytes": 4 * nkv * (total + B * width + B * case["budget"]) + 8 * nkv * dim * kept, "flops": nkv * total}


# ------------------------------------------------------------------ the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


def _exact_logprobs(s):
    top, vocab = s["case"]["top"], s["case"]["vocab"]
    lp, entropy, top_lp, top_ids = [], [], [], []
    for z, t in zip(s["logits"], s["targets"].tolist()):
        z = z.double()
        logp = z - torch.logsumexp(z, 0)
        lp.append(logp[t] if t >= 0 else logp.new_zeros(()))
        p = logp.exp()
        entropy.append(-(p[p > 0] * logp[p > 0]).sum())
        if top:
            i = torch.argsort(z, descending=True, stable=True)[:top]
            top_ids.append(i)
            top_lp.append(logp[i])
    if not top:
        return torch.stack(lp), torch.stack(entropy)
    return torch.stack(lp), torch.stack(entropy), torch.stack(top_lp), torch.stack(top_ids)


def _exact_append(s):
    case = s["case"]
    nq, nkv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    half = dim // 2
    k, v = s["k"].double(), s["v"].double()
    x = s["qkv"].double().unflatten(1, (nq + 2 * nkv, dim))
    p = s["positions"].long()
    c, d = s["cos"].double()[p].unsqueeze(1), s["sin"].double()[p].unsqueeze(1)
    rot = torch.empty_like(x)
    rot[..., :half] = x[..., :half] * c[..., :half] - x[..., half:] * d[..., :half]
    rot[..., half:] = x[..., half:] * c[..., half:] + x[..., :half] * d[..., half:]
    pages = s["table"].long()[s["seqs"].long(), torch.div(s["slots"].long(), page, rounding_mode="floor")]
    row = s["slots"].long().remainder(page)
    for h in range(nkv):
        k[pages, h, row] = rot[:, nq + h]
        v[pages, h, row] = x[:, nq + nkv + h]
    return rot[:, :nq], k, v


def _exact_attend(s):
    case = s["case"]
    B, nq, nkv, dim, page = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = nq // nkv
    out = torch.zeros(B, nq, dim, device="cuda", dtype=torch.float64)
    weights = s["weights"].double() if case["weights"] else None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        mine = s["table"][b, : _pages(n, case)].long()
        for h in range(nkv):
            k = s["k"][mine, h].reshape(-1, dim)[:n].double()
            v = s["v"][mine, h].reshape(-1, dim)[:n].double()
            p = torch.softmax(s["q"][b, h * group: (h + 1) * group].double() @ k.T / math.sqrt(dim), -1)
            out[b, h * group: (h + 1) * group] = p @ v
            if weights is not None:
                weights[b, h, :n] += p.sum(0)
    return (out, weights) if case["weights"] else (out,)


def _exact_evict(s):
    case = s["case"]
    B, nkv, page, budget = case["seqs"], case["kv_heads"], case["page"], case["budget"]
    k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
    new_w = torch.zeros_like(w)
    for b, n in enumerate(s["lens"].tolist()):
        m = min(n, budget)
        old = max(0, n - case["recent"])
        to = torch.arange(m, device="cuda")
        to_page = s["new_table"][b].long()[to // page]
        for h in range(nkv):
            if m == n:
                keep = to
            else:
                best = torch.argsort(w[b, h, :old], descending=True, stable=True)[: m - (n - old)]
                keep = torch.cat([best.sort().values, torch.arange(old, n, device="cuda")])
            new_w[b, h, :m] = w[b, h, keep]
            at = s["table"][b].long()[keep // page]
            k[to_page, h, to % page] = k[at, h, keep % page]
            v[to_page, h, to % page] = v[at, h, keep % page]
    return None, None, new_w, k, v
