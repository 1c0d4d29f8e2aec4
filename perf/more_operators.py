"""Performance cases of dense attention over a paged cache, and of what a model answers.

Every case is one pass through operators of nanokv_amd.paged or nanokv_amd.logprobs:

  append    the fused projection's rows: norms of queries and keys (or none),
            the rotation of their positions, keys and values written to their slots
            of a paged cache in bf16 or 8 bits (qkv_append_paged; read_paged
            reads 8-bit slots back);
  attend    attention of new tokens over a paged cache: one token a sequence,
            a tree of drafted tokens, prompts (attend_paged);
  logprobs  log probabilities of given tokens, the entropy of their distribution
            and its most likely alternatives (token_logprobs).

With `own` false `run` computes them in elementary torch operations, in 32 bits.
`exact` restates each of them in 64 bits.
"""

import math
import os
import sys

import torch

own = False

EPS = 1e-6
BASE = 1000000.0
MOST_PAIRS = 32 * 128 * 4096 * (12288 + 2048)    # head dims * (query, key) pairs of the largest attention
MOST_CACHE = 64 * 4096 * 8 * 128                 # elements of keys of the largest cache
MOST_LOGITS = 2048 * 151936


def listed():
    return [
        # one decode token of one sequence: the smallest call
        {"name": "append_token", "op": "append", "rows": 1, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "norm": True, "kv": "bf16", "page": 64},
        # one decode token of each of many sequences, the cache in 8 bits, a few rows of padding
        {"name": "append_batch_96_int8", "op": "append", "rows": 96, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "norm": True, "kv": "int8", "page": 64},
        # a default prompt chunk
        {"name": "append_chunk", "op": "append", "rows": 4096, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "norm": True, "kv": "bf16", "page": 256},
        # a ragged prompt of a model without norms that rotates neighbouring pairs of half of each head
        {"name": "append_pairs_1777", "op": "append", "rows": 1777, "hq": 16, "hkv": 8, "d": 128, "rot": 64,
         "interleaved": True, "norm": False, "kv": "bf16", "page": 16},
        # one token of one short sequence
        {"name": "attend_token", "op": "attend", "batch": 1, "new": 1, "context": 2048, "hq": 32, "hkv": 8, "d": 128,
         "kv": "bf16", "page": 64, "tree": False},
        # one token of each of 64 sequences of unequal length
        {"name": "attend_batch_64", "op": "attend", "batch": 64, "new": 1, "context": 8192, "hq": 32, "hkv": 8,
         "d": 128, "kv": "bf16", "page": 64, "tree": False},
        # one token of three very long sequences in 8 bits
        {"name": "attend_long_int8", "op": "attend", "batch": 3, "new": 1, "context": 131072, "hq": 32, "hkv": 8,
         "d": 128, "kv": "int8", "page": 64, "tree": False},
        # a tree of drafted tokens in each of five sequences
        {"name": "attend_tree_26", "op": "attend", "batch": 5, "new": 26, "context": 16384, "hq": 32, "hkv": 8,
         "d": 128, "kv": "bf16", "page": 64, "tree": True},
        # a batch of whole prompts of unequal length, small heads
        {"name": "attend_prompts", "op": "attend", "batch": 7, "new": 2000, "context": 0, "hq": 16, "hkv": 8, "d": 64,
         "kv": "bf16", "page": 16, "tree": False},
        # a default prompt chunk behind an older part of its prompt: the largest call
        {"name": "attend_chunk", "op": "attend", "batch": 1, "new": 4096, "context": 12288, "hq": 32, "hkv": 8,
         "d": 128, "kv": "bf16", "page": 256, "tree": False},
        # the answer's next token, with 20 alternatives
        {"name": "logprobs_token", "op": "logprobs", "rows": 1, "vocab": 151936, "dtype": "float32", "top": 20,
         "masked": False},
        # the tokens of a prompt
        {"name": "logprobs_prompt", "op": "logprobs", "rows": 2048, "vocab": 151936, "dtype": "bfloat16", "top": 5,
         "masked": False},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = log_int(1000, 160000)
        rows = rng.choice([1, rng.randint(2, 16), log_int(17, 2048)])
        return {"op": op, "rows": max(1, min(rows, MOST_LOGITS // vocab)), "vocab": vocab,
                "dtype": rng.choice(["float32", "bfloat16"]) if rows < 1024 else "bfloat16",
                "top": rng.choice([1, 5, 20, 50]), "masked": rng.random() < 0.3}
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8, 8])
    hq = hkv * rng.choice([1, 2, 4, 4, 5, 8])
    case = {"op": op, "hq": hq, "hkv": hkv, "d": d, "kv": rng.choice(["bf16", "bf16", "int8"]),
            "page": rng.choice([16, 32, 64, 128, 256])}
    if op == "append":
        rot = rng.choice([d, d, d // 2])
        case.update(rows=rng.choice([1, rng.randint(2, 128), log_int(129, 4096)]), rot=rot,
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.6)
        return case
    kind = rng.choice(["token", "token", "tree", "prompt"])
    if kind == "token":
        batch, new, context = log_int(1, 128), 1, log_int(64, 131072)
    elif kind == "tree":
        batch, new, context = log_int(1, 16), rng.randint(2, 64), log_int(64, 32768)
    else:
        batch, new, context = rng.randint(1, 8), log_int(100, 4096), rng.choice([0, log_int(64, 16384)])
    while batch * (context + new) * hkv * d > MOST_CACHE:
        context = context // 2
    while batch * new * (context + new // 2) * hq * d > MOST_PAIRS:
        new = new * 3 // 4
    case.update(batch=batch, new=max(1, new), context=context, tree=kind == "tree")
    return case


# -- inputs ------------------------------------------------------------------
def _lengths(case):
    """(keys, new tokens) of every sequence: from the largest down to a tenth, in no order."""
    b, new, context = case["batch"], case["new"], case["context"]
    part = [1.0 if i == b // 2 else 0.1 + 0.9 * ((0.37 + 0.6180339887 * i) % 1.0) for i in range(b)]
    count = [new if new == 1 or case["tree"] else max(1, int(new * p)) for p in part]
    return [int(context * p) + n for p, n in zip(part, count)], count


def _parents(n, rng_row):
    """A tree of n drafted tokens: each hangs on one of those before it (-1: on the cache)."""
    return [-1] + [min(i - 1, int(r * i)) - (1 if i < 4 else 0) for i, r in zip(range(1, n), rng_row)]


def _tables(rot, positions, device="cuda"):
    ang = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * (
        BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot))
    return ang.cos().float(), ang.sin().float()


def _cache(g, pages, hkv, page, d, kv):
    """Keys and values of a paged cache [pages, hkv, page, d], scales [pages, hkv, page] in 8 bits."""
    shape = (pages, hkv, page, d)
    if kv == "int8":
        return {n: torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for n in "kv"} | {
            n + "s": torch.rand(shape[:3], generator=g, device="cuda") * 0.02 + 0.005 for n in "kv"}
    cache = {}
    for n in "kv":
        cache[n] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        for part in cache[n].split(max(1, (1 << 26) // (hkv * page * d))):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return cache | {"ks": None, "vs": None}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)
    op = case["op"]
    if op == "logprobs":
        return _prepare_logits(case, g)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    if op == "append":
        rows = case["rows"]
        pages = -(-rows // page) + 2
        # a sequence's slots run on from page to page of a table in no order; a few rows of padding
        order = torch.randperm(pages - 1, generator=g, device="cuda")
        at = torch.arange(rows, device="cuda") + 3
        slots = (order[at // page] * page + at % page).to(torch.int32)
        if rows > 16:
            slots[-(rows // 16):] = -1
        s = {"op": op, "slots": slots, "page": page, "hq": hq, "hkv": hkv, "interleaved": case["interleaved"],
             "spare": (pages - 1) * page}
        ch = torch.randn((hq + 2 * hkv) * d, generator=g, device="cuda").mul_(0.5).exp_()
        s["qkv"] = (torch.randn(rows, (hq + 2 * hkv) * d, generator=g, device="cuda") * ch).to(torch.bfloat16)
        first = int(seed) % 20000
        s["positions"] = torch.arange(first, first + rows, device="cuda")
        s["cos"], s["sin"] = _tables(case["rot"], 40960)
        for n in ("q_norm", "k_norm"):
            s[n] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16) if case["norm"] else None
        return s | _cache(g, pages, hkv, page, d, case["kv"])
    keys, count = _lengths(case)
    b, most = len(keys), max(-(-n // page) for n in keys)
    total = sum(-(-n // page) for n in keys)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros(b, most, dtype=torch.int32, device="cuda")
    used = 0
    for i, n in enumerate(keys):
        own_pages = -(-n // page)
        tables[i, :own_pages] = order[used:used + own_pages]
        used += own_pages
    starts = [0]
    for n in count:
        starts.append(starts[-1] + n)
    s = {"op": op, "page": page, "hkv": hkv, "scale": d ** -0.5, "tables": tables, "max_new": max(count),
         "lengths": torch.tensor(keys, dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda") if case["new"] > 1 else None, "tree": None}
    s["q"] = (torch.randn(starts[-1], hq, d, generator=g, device="cuda") * 1.5).to(torch.bfloat16)
    if case["tree"]:
        n = case["new"]
        draws = torch.rand(b, n, generator=g, device="cuda").tolist()
        masks = []
        for row in draws:
            seen = []
            for i, p in enumerate(_parents(n, row)):
                m = (1 << i) | (seen[p] if p >= 0 else 0)
                seen.append(m)
            masks += [m - (1 << 64) if m >= 1 << 63 else m for m in seen]
        s["tree"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
    return s | _cache(g, total, hkv, page, d, case["kv"])


def _prepare_logits(case, g):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    x = torch.empty(rows, vocab, dtype=getattr(torch, case["dtype"]), device="cuda")
    for part in x.split(max(1, (1 << 26) // vocab)):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * 2.2)
    likely = torch.randint(0, vocab, (rows, 40), generator=g, device="cuda")
    x.scatter_(1, likely, (torch.randn(rows, 40, generator=g, device="cuda") * 3 + 11).to(x.dtype))
    if case["masked"]:      # a grammar that allows about one token in four
        x.masked_fill_(torch.rand(vocab, generator=g, device="cuda") < 0.75, float("-inf"))
    pick = torch.randint(0, 40, (rows, 1), generator=g, device="cuda")
    return {"op": "logprobs", "logits": x, "tokens": likely.gather(1, pick)[:, 0], "top": top}


# -- the plain form ----------------------------------------------------------
def _rotated(x, cos, sin, interleaved):
    """x [rows, heads, d] fp32, its first 2 * cos.shape[-1] dims rotated."""
    r = 2 * cos.shape[-1]
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _normed(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()


def _plain_append(s):
    hq, hkv, page = s["hq"], s["hkv"], s["page"]
    x = s["qkv"].float()
    x = x.view(x.shape[0], hq + 2 * hkv, -1)
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _rotated(_normed(x[:, :hq], s["q_norm"]), cos, sin, s["interleaved"])
    k = _rotated(_normed(x[:, hq:hq + hkv], s["k_norm"]), cos, sin, s["interleaved"])
    new = {"k": k, "v": x[:, hq + hkv:]}
    live = s["slots"] >= 0
    slots = torch.where(live, s["slots"], s["spare"]).long()
    p, o = slots // page, slots % page
    out = {"q": q.to(torch.bfloat16)}
    for n, y in new.items():
        held = s[n]
        if s[n + "s"] is None:
            held[p, :, o] = torch.where(live[:, None, None], y.to(torch.bfloat16), held[p, :, o])
            out[n] = held
        else:
            top = y.abs().amax(dim=-1, keepdim=True)
            codes = torch.round(y * (127.0 / top))
            held[p, :, o] = torch.where(live[:, None, None], codes.to(torch.int8), held[p, :, o])
            s[n + "s"][p, :, o] = torch.where(live[:, None], top[..., 0] / 127.0, s[n + "s"][p, :, o])
            out[n] = torch.where(live[:, None, None], codes * (top / 127.0), 0.0).to(torch.bfloat16)
    return out


def _gathered(s, n):
    """fp32 [batch, hkv, keys, d] of the cache's keys or values, padded to the longest table."""
    x = s[n][s["tables"].long()].float()          # [batch, pages, hkv, page, d]
    if s[n + "s"] is not None:
        x = x * s[n + "s"][s["tables"].long()].unsqueeze(-1)
    return x.transpose(1, 2).flatten(2, 3)


def _visible(s, b, n, keys):
    """bool [batch, n, keys]: the keys that query i of a sequence sees (queries past its last see none)."""
    dev = s["q"].device
    length = s["lengths"].long()[:, None, None]
    j = torch.arange(keys, device=dev)
    i = torch.arange(n, device=dev)[:, None]
    if s["starts"] is None:
        return j < length
    begin = s["starts"].long()[:-1, None, None]
    count = s["starts"].long()[1:, None, None] - begin
    older = length - count
    if s["tree"] is None:
        return (j <= older + i) & (i < count)
    rows = (begin[:, :, 0] + i[:, 0]).clamp(max=s["q"].shape[0] - 1)
    bits = s["tree"][rows][:, :, None] >> (j - older).clamp(0, 63)
    return ((j < older) | ((j < length) & (bits & 1).bool())) & (i < count)


def _plain_attend(s):
    q = s["q"].float()
    rows, hq, d = q.shape
    b, n, hkv = s["lengths"].shape[0], s["max_new"], s["hkv"]
    g = hq // hkv
    k, v = _gathered(s, "k"), _gathered(s, "v")
    seen = _visible(s, b, n, k.shape[2])
    first = torch.arange(b, device=q.device) if s["starts"] is None else s["starts"].long()[:-1]
    at = (first[:, None] + torch.arange(n, device=q.device)).clamp(max=rows - 1)
    # [batch, hkv, queries * heads of a key head, d]
    qs = q[at].view(b, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    w = qs @ k.transpose(-1, -2)
    w = w.view(b, hkv, n, g, -1).mul_(s["scale"]).masked_fill_(~seen[:, None, :, None], float("-inf"))
    w = w.sub_(w.amax(dim=-1, keepdim=True).nan_to_num(neginf=0.0)).exp_()
    total = w.sum(dim=-1, keepdim=True)
    o = (w.view(b, hkv, n * g, -1) @ v).view(b, hkv, n, g, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)
    if s["starts"] is None:
        return o.view(rows, hq, d).to(torch.bfloat16)
    row = torch.arange(rows, device=q.device)
    seq = torch.searchsorted(s["starts"].long()[1:], row, right=True)
    return o[seq, row - first[seq]].to(torch.bfloat16)


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(dim=-1, keepdim=True)
    y = x - m
    e = y.exp()
    total = e.sum(dim=-1)
    log_total = total.log()
    terms = torch.where(e > 0, y * e, 0.0).sum(dim=-1)
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    values, ids = values[:, :s["top"]], ids[:, :s["top"]]
    return {"logprob": y.gather(1, s["tokens"][:, None])[:, 0] - log_total, "entropy": log_total - terms / total,
            "top_logprobs": values - m - log_total[:, None], "top_ids": ids.contiguous()}


# -- the framework -------------------------------------------------------------
def _framework():
    """nanokv_amd's modules, imported once as a program does, not in every pass."""
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-kv-optimizer_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from nanokv_amd import logprobs, paged
    return paged, logprobs


def _own(s):
    paged, logprobs = sys.modules.get("nanokv_amd.paged"), sys.modules.get("nanokv_amd.logprobs")
    if paged is None or logprobs is None:
        paged, logprobs = _framework()
    if s["op"] == "logprobs":
        t = logprobs.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return {"logprob": t.logprob, "entropy": t.entropy, "top_logprobs": t.top_logprobs, "top_ids": t.top_ids}
    cache = paged.PagedKV(s["k"], s["v"], s["ks"], s["vs"])
    if s["op"] == "attend":
        return paged.attend_paged(s["q"], cache, s["tables"], s["lengths"], starts=s["starts"], max_new=s["max_new"],
                                  tree=s["tree"], scale=s["scale"])
    q = paged.qkv_append_paged(cache, s["qkv"], s["slots"], s["positions"], s["cos"], s["sin"], s["hq"],
                               q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, interleaved=s["interleaved"])
    if s["ks"] is None:
        return {"q": q, "k": s["k"], "v": s["v"]}
    k, v = paged.read_paged(cache, s["slots"])
    return {"q": q, "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "append":
        return _plain_append(state)
    if state["op"] == "attend":
        return _plain_attend(state)
    return _plain_logprobs(state)


# -- what a pass cannot do without -------------------------------------------
def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * n}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    row = d + 4 if case["kv"] == "int8" else 2 * d        # a held key or value of one head
    if case["op"] == "append":
        rows = case["rows"]
        live = rows - (rows // 16 if rows > 16 else 0)
        b = rows * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 12 + 4 * case["rot"]) + live * 2 * hkv * row
        if case["kv"] == "int8":                         # and read back
            b += live * 2 * hkv * row + rows * 2 * hkv * d * 2
        return {"bytes": b, "flops": rows * d * (8 * (hq + hkv) + (8 * hkv if case["kv"] == "int8" else 0))}
    keys, count = _lengths(case)
    pairs = sum(n * (k - n) + (n * (n + 1) // 2) for k, n in zip(keys, count))
    return {"bytes": sum(keys) * hkv * 2 * row + 4 * sum(count) * hq * d + 4 * sum(-(-k // case["page"]) for k in keys),
            "flops": 4 * d * hq * pairs}


# -- in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s, case)
    return (_exact_append if case["op"] == "append" else _exact_attend)(s, case)


def _exact_append(s, case):
    hq, hkv, d, page, rot = case["hq"], case["hkv"], case["d"], case["page"], case["rot"]
    x = s["qkv"].double().reshape(-1, hq + 2 * hkv, d)

    def turn(part, weight):
        y = part
        if weight is not None:
            y = y / (y.square().sum(dim=2, keepdim=True) / d + EPS).sqrt() * weight.double()
        first = torch.arange(0, rot, 2, device=y.device) if case["interleaved"] else torch.arange(rot // 2, device=y.device)
        second = first + (1 if case["interleaved"] else rot // 2)
        z = torch.complex(y[..., first], y[..., second]) * torch.complex(
            s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]).unsqueeze(1)
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"q": turn(x[:, :hq], s["q_norm"])}
    for n, y in (("k", turn(x[:, hq:hq + hkv], s["k_norm"])), ("v", x[:, hq + hkv:])):
        keep = (s["slots"] >= 0).nonzero()[:, 0]
        if case["kv"] == "int8":
            step = y.abs().max(dim=2, keepdim=True).values / 127.0
            held = torch.zeros_like(y)
            held[keep] = ((y / step).round() * step)[keep]
        else:
            held = s[n].double()
            at = s["slots"].long()[keep]
            held[torch.div(at, page, rounding_mode="floor"), :, at % page] = y[keep]
        out[n] = held
    return out


def _exact_attend(s, case):
    keys, count = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    g, out, at = hq // hkv, [], 0
    for b, (length, n) in enumerate(zip(keys, count)):
        pages = s["tables"][b, :-(-length // page)].long()
        older = length - n
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if case["tree"]:
            bit = torch.arange(n, device="cuda")
            seen[:, older:] = ((s["tree"][at:at + n, None] >> bit) & 1).bool()
        else:
            seen = seen.tril(older)
        heads = []
        for h in range(hkv):
            kv = []
            for name in "kv":
                t = s[name][pages, h].double()
                if case["kv"] == "int8":
                    t = t * s[name + "s"][pages, h].double().unsqueeze(-1)
                kv.append(t.reshape(-1, d)[:length])
            for e in range(g):
                logits = s["q"][at:at + n, h * g + e].double() @ kv[0].t() * s["scale"]
                logits[~seen] = float("-inf")
                heads.append(torch.softmax(logits, dim=1) @ kv[1])
        out.append(torch.stack(heads, dim=1))
        at += n
    return torch.cat(out)


def _exact_logprobs(s, case):
    parts = []
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        lp = torch.log_softmax(x, dim=1)
        h = -torch.where(lp > float("-inf"), lp.exp() * lp, 0.0).sum(dim=1)
        best = torch.topk(lp, case["top"], dim=1).values
        parts.append((lp.gather(1, t.unsqueeze(1)).squeeze(1), h, best))
    lp, h, best = (torch.cat(p) for p in zip(*parts))
    return {"logprob": lp, "entropy": h, "top_logprobs": best, "top_ids": None}
