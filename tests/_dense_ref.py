"""Float64 restatement of the Qwen3 decoder with dense causal attention over one whole sequence."""

import torch


def dense_logits(model, ids):
    """Logits [T, vocab] of ids [T] (a path of a drafted tree is a sequence of its own)."""
    c, w = model.config, {k: v.detach().double().cpu() for k, v in model.state_dict().items()}
    T, hq, hkv, d = len(ids), c.num_attention_heads, c.num_key_value_heads, c.head_dim
    ids = torch.as_tensor(ids).cpu()
    ang = torch.arange(T).double()[:, None, None] * (
        c.rope_theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    cos, sin = ang.cos(), ang.sin()

    def rms(x, g):
        return x / (x.pow(2).mean(-1, keepdim=True) + c.rms_norm_eps).sqrt() * g

    def rope(x):
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    r = w["model.embed_tokens.weight"][ids]
    for i in range(c.num_hidden_layers):
        p = f"model.layers.{i}."
        qkv = rms(r, w[p + "input_layernorm.weight"]) @ w[p + "self_attn.qkv_proj.weight"].T
        if c.attention_bias:
            qkv = qkv + w[p + "self_attn.qkv_proj.bias"]
        q, k, v = (x.reshape(T, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], -1))
        if not c.attention_bias:
            q, k = rms(q, w[p + "self_attn.q_norm.weight"]), rms(k, w[p + "self_attn.k_norm.weight"])
        q, k = rope(q), rope(k)
        s = torch.einsum("thgd,shd->hgts", q.view(T, hkv, hq // hkv, d), k) * d ** -0.5
        s = s.masked_fill(torch.ones(T, T).triu(1).bool(), float("-inf")).softmax(-1)
        o = torch.einsum("hgts,shd->thgd", s, v).reshape(T, hq * d)
        r = r + o @ w[p + "self_attn.o_proj.weight"].T
        g, u = (rms(r, w[p + "post_attention_layernorm.weight"]) @ w[p + "mlp.gate_up_proj.weight"].T).chunk(2, -1)
        r = r + (g * torch.sigmoid(g) * u) @ w[p + "mlp.down_proj.weight"].T
    return rms(r, w["model.norm.weight"]) @ w["lm_head_weight"].T


def one_step(model, device, kv, ids):
    """Logits [T, vocab] of one sequence in one step over a cache of its own."""
    pages = -(-len(ids) // 16)
    model.attach_paged(pages, 16, torch.int8 if kv == "int8" else torch.bfloat16)
    at = torch.arange(len(ids), device=device)
    h = model.paged_step(torch.as_tensor(ids, device=device), at, at, torch.arange(pages, device=device)[None],
                         torch.tensor([len(ids)], device=device),
                         starts=torch.tensor([0, len(ids)], device=device))
    return model.compute_logits(h)


def serve(model, device, kv, check):
    """A run as a server makes it, three sequences at once: prompts of unequal length (one in two
    chunks), a token each, a drafted tree each, its accepted path moved up, a token behind it.
    check(name, hidden rows, [the sequence that each row ends]) after every step."""
    from nanokv_amd.paged import move_paged, tree_masks
    caches = model.attach_paged(24, 16, torch.int8 if kv == "int8" else torch.bfloat16)
    g = torch.Generator().manual_seed(2)
    ids = [torch.randint(0, model.config.vocab_size, (n,), generator=g).tolist() for n in (37, 5, 70)]
    order = torch.randperm(24, generator=g).view(3, 8).to(torch.int32)
    tables = order.to(device)

    def slots(b, places):
        return [int(order[b, p // 16]) * 16 + p % 16 for p in places]

    def step(tokens, places, keys, parents=None):
        """Each sequence's new tokens at its places (the cache's), `keys` keys with them."""
        n = [len(t) for t in tokens]
        starts = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32, device=device)
        depth = [list(p) for p in places]
        tree = None
        if parents is not None:
            tree = torch.cat([tree_masks(torch.tensor(p)) for p in parents]).to(device)
            for b, p in enumerate(parents):        # a drafted token's position is its depth behind the sequence
                depth[b] = []
                for i, q in enumerate(p):
                    depth[b].append(places[b][0] if q < 0 else depth[b][q] + 1)
        flat = lambda rows: torch.tensor([x for r in rows for x in r], device=device)  # noqa: E731
        return model.paged_step(flat(tokens), flat(depth), flat([slots(b, p) for b, p in enumerate(places)]), tables,
                                torch.tensor(keys, dtype=torch.int32, device=device),
                                starts=None if max(n) == min(n) == 1 else starts, max_new=max(n), tree=tree)

    first = [37, 5, 41]
    h = step([s[:n] for s, n in zip(ids, first)], [range(n) for n in first], first)
    check("prompts", h, [s[:i + 1] for s, n in zip(ids, first) for i in range(n)])
    h = step([[7], [8], ids[2][41:]], [[37], [5], range(41, 70)], [38, 6, 70])
    seq = [ids[0] + [7], ids[1] + [8], ids[2]]
    check("tokens and a chunk", h, [seq[0], seq[1]] + [seq[2][:i + 1] for i in range(41, 70)])
    tokens = [[11], [12], [13]]
    h = step(tokens, [[len(s)] for s in seq], [len(s) + 1 for s in seq])
    seq = [s + t for s, t in zip(seq, tokens)]
    check("tokens", h, seq)
    parents = [[-1, 0, 0, 1, 2, 4], [-1, -1, 1], [-1, 0, 1, 1, 0, 4, 5]]
    drafts = [[20 + i for i in range(len(p))] for p in parents]
    h = step(drafts, [range(len(s), len(s) + len(p)) for s, p in zip(seq, parents)],
             [len(s) + len(p) for s, p in zip(seq, parents)], parents)
    paths = []
    for p in parents:
        paths.append([])
        for i, q in enumerate(p):
            paths[-1].append((paths[-1][q] if q >= 0 else []) + [i])
    check("trees", h, [s + [d[i] for i in path] for s, d, ps in zip(seq, drafts, paths) for path in ps])
    taken = [ps[i] for ps, i in zip(paths, (5, 2, 3))]       # what the target accepts of each tree
    src = [x for b, t in enumerate(taken) for x in slots(b, [len(seq[b]) + i for i in t])]
    dst = [x for b, t in enumerate(taken) for x in slots(b, range(len(seq[b]), len(seq[b]) + len(t)))]
    for cache in caches:
        move_paged(cache, torch.tensor(src, device=device), torch.tensor(dst, device=device))
    seq = [s + [d[i] for i in t] for s, d, t in zip(seq, drafts, taken)]
    h = step([[40], [41], [42]], [[len(s)] for s in seq], [len(s) + 1 for s in seq])
    check("behind the accepted paths", h, [s + [40 + b] for b, s in enumerate(seq)])
