"""The paged KV cache operators in float64 torch, one sequence at a time."""
import math

import torch


def make(seed, dtype, new, past, heads, kv_heads, head, page, shared=0, device="cuda",
         spare_pages=2, garbage=True):
    """A ragged batch: caches whose unused rows hold NaN (when `garbage`),
    pages in random order, the first `shared` positions in common."""
    g = torch.Generator().manual_seed(seed)
    total = [n + p for n, p in zip(new, past)]
    pages = [-(-t // page) for t in total]
    order = torch.randperm(sum(pages) + spare_pages, generator=g).to(torch.int32)
    table = torch.full((len(new), max(pages + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    whole = shared // page
    shape = (sum(pages) + spare_pages, page, kv_heads, head)
    key = torch.full(shape, math.nan if garbage else 0.0)
    value = key.clone()
    pre = [torch.randn((shared, kv_heads, head), generator=g) for _ in range(2)]
    for b, t in enumerate(total):
        if t:
            table[b, :whole] = table[0, :whole]
            pos = torch.arange(t)
            where = (table[b][pos // page].long(), pos % page)
            for i, cache in enumerate((key, value)):
                x = torch.randn((t, kv_heads, head), generator=g)
                x[:shared] = pre[i]
                cache[where] = x
    cu = torch.zeros(len(new) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(new).cumsum(0)
    return dict(key=key.to(dtype).to(device), value=value.to(dtype).to(device),
                table=table.to(device), cu=cu.to(device),
                past=torch.tensor(past, dtype=torch.int32).to(device),
                q=torch.randn((sum(new), heads * head), generator=g).to(device))


def attention(s, new, past, heads, scale=None, softcap=0.0, window=0):
    """softmax(cap(scale q.k)) v over the visible keys, in float64."""
    G, D = s["key"].shape[2:]
    page = s["key"].shape[1]
    out = torch.zeros((sum(new), heads, D), dtype=torch.float64, device=s["q"].device)
    row = 0
    for b, (n, p0) in enumerate(zip(new, past)):
        pos = torch.arange(n + p0, device=out.device)
        where = (s["table"][b][pos // page].long(), pos % page)
        k, v = s["key"][where].double(), s["value"][where].double()
        for i in range(n):
            lo = max(0, p0 + i + 1 - window) if window else 0
            hi = p0 + i + 1
            q = s["q"][row].double().view(G, heads // G, D)
            sc = torch.einsum("ghd,tgd->ght", q, k[lo:hi]) * (scale or 1 / math.sqrt(D))
            if softcap:
                sc = softcap * torch.tanh(sc / softcap)
            out[row] = torch.einsum("ght,tgd->ghd", torch.softmax(sc, -1), v[lo:hi]).reshape(
                heads, D)
            row += 1
    return out.view(sum(new), heads * D)


def rotate(x, cos, sin, interleaved):
    """RoPE of x [tokens, heads, head] by cos/sin [tokens, half], float64."""
    half = cos.shape[-1]
    y = x.double().clone()
    c, z = cos.double()[:, None], sin.double()[:, None]
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    x0, x1 = y[..., a].clone(), y[..., b].clone()
    y[..., a] = x0 * c - x1 * z
    y[..., b] = x1 * c + x0 * z
    return y
