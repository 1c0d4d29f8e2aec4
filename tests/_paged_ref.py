"""A paged cache's operators restated in 64 bits, for the tests."""

import torch


def make_cache(pages, hkv, page, d, kv, device, seed=0, fill=None):
    """A PagedKV of random rows (or of `fill` everywhere)."""
    from nanokv_amd.paged import PagedKV
    g = torch.Generator().manual_seed(seed)
    shape = (pages, hkv, page, d)
    if kv == "int8":
        codes = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).to(device) for _ in range(2)]
        scales = [(torch.rand(shape[:3], generator=g) * 0.02 + 0.005).to(device) for _ in range(2)]
        return PagedKV(*codes, *scales)
    if fill is not None:
        return PagedKV(*(torch.full(shape, fill, dtype=torch.bfloat16, device=device) for _ in range(2)))
    return PagedKV(*(torch.randn(shape, generator=g).bfloat16().to(device) for _ in range(2)))


def held(cache, which):
    """Values of the cache's keys (0) or values (1) in 64 bits: [pages, hkv, page, d]."""
    x = cache[which].double()
    return x if cache[2 + which] is None else x * cache[2 + which].double().unsqueeze(-1)


def rope_tables(positions, rot, device, base=10000.0):
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return ang.cos().float().to(device), ang.sin().float().to(device)


def heads_ref(x, weight, eps, cos, sin, interleaved):
    """(x normed and rotated, the magnitude of the terms each value is the sum of), 64 bits;
    x [T, heads, d], cos, sin [T, R / 2] or None."""
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    mag = y.abs()
    if cos is None:
        return y, mag
    r = 2 * cos.shape[1]
    a = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    b = a + (1 if interleaved else r // 2)
    a, b = a.to(x.device), b.to(x.device)
    c, s = cos.double()[:, None], sin.double()[:, None]
    out, size = y.clone(), mag.clone()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    size[..., a] = (y[..., a] * c).abs() + (y[..., b] * s).abs()
    size[..., b] = (y[..., b] * c).abs() + (y[..., a] * s).abs()
    return out, size


def attend_ref(q, cache, tables, lengths, starts=None, tree=None, scale=None, n_each=1):
    """Attention of every row in 64 bits, key by key; (out, sum of p |v|) [T, hq, d].

    Hidden keys are left out, not weighted with 0; rows that see nothing, and rows of no
    sequence, are 0."""
    T, hq, d = q.shape
    hkv, page = cache.k.shape[1], cache.k.shape[2]
    pages = cache.k.shape[0]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    q, k, v = q.double().cpu(), held(cache, 0).cpu(), held(cache, 1).cpu()
    tables, lengths = tables.cpu(), lengths.cpu()
    B = lengths.shape[0]
    starts = [b * n_each for b in range(B + 1)] if starts is None else starts.cpu().tolist()
    tree = None if tree is None else tree.cpu().tolist()
    out, mag = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    for b in range(B):
        n, L = starts[b + 1] - starts[b], min(int(lengths[b]), tables.shape[1] * page)
        ids = [int(tables[b, j // page]) for j in range(L)]
        ok = torch.tensor([0 <= p < pages for p in ids], dtype=torch.bool)
        at = torch.tensor([max(0, min(p, pages - 1)) for p in ids], dtype=torch.long)
        off = torch.arange(L) % page
        older = L - n
        keys, values = k[at, :, off], v[at, :, off]                            # [L, hkv, d]
        for i in range(n):
            t = starts[b] + i
            seen = torch.arange(L) <= older + i
            if tree is not None:
                m = tree[t] & ((1 << 64) - 1)
                seen = torch.tensor([j < older or (0 <= j - older < 64 and bool(m >> (j - older) & 1)) for j in range(L)],
                                    dtype=torch.bool)
            seen &= ok
            if not bool(seen.any()):
                continue
            kk, vv = keys[seen], values[seen]
            qq = q[t].view(hkv, g, d)
            w = torch.softmax(torch.einsum("hgd,khd->hgk", qq, kk) * scale, dim=-1)
            out[t] = torch.einsum("hgk,khd->hgd", w, vv).reshape(hq, d)
            mag[t] = torch.einsum("hgk,khd->hgd", w, vv.abs()).reshape(hq, d)
    return out, mag
