"""The quantised cache's operators from their definitions, in Python and 64 bits
on the CPU: the page table step, the quantising append and the attention.
Test infrastructure, written for reading: loops over requests, runs and heads."""
import math

import torch

CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOOR = 2.0 ** -100


def page_table_step(table, before, after, free, num_free, page_size, total_new, idx=None):
    """Lists in, (table, free, slots, cu, num_free_out) out."""
    table, free = [list(r) for r in table], list(free)
    width = len(table[0]) if table else 0
    top = min(max(num_free, 0), len(free))
    rows = [b if idx is None else idx[b] for b in range(len(before))]
    rows = [r if 0 <= r < len(table) else None for r in rows]
    pages = lambda n: min(-(-max(n, 0) // page_size), width)  # noqa: E731
    for r, x, y in zip(rows, before, after):
        if r is None:
            continue
        for j in range(pages(y), pages(x)):
            if table[r][j] >= 0 and top < len(free):
                free[top] = table[r][j]
                top += 1
    slots, cu = [], [0]
    for r, x, y in zip(rows, before, after):
        if r is not None:
            for j in range(pages(x), pages(y)):
                top -= 1
                table[r][j] = free[top] if top >= 0 else -1
        for at in range(max(x, 0), max(y, 0)):
            j = at // page_size
            ok = r is not None and j < width and table[r][j] >= 0
            slots.append(table[r][j] * page_size + at % page_size if ok else -1)
        cu.append(len(slots))
    slots = (slots + [-1] * total_new)[:total_new]
    return table, free, slots, cu, top


def encode(x, dtype):
    """Codes of the 64-bit x: nearest, ties to even."""
    if dtype == torch.int8:
        return torch.round(torch.nan_to_num(x, nan=0.0).clamp(-127, 127)).to(torch.int8)
    # e4m3: 3 bits behind the leading one, at least 2 ** -9 apart, 448 the largest
    m, e = torch.frexp(torch.nan_to_num(x, nan=0.0).clamp(-448, 448))
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 4, min=-9))
    y = torch.round(torch.nan_to_num(x, nan=0.0).clamp(-448, 448) / step) * step
    return torch.where(torch.isnan(x), torch.nan, y).float().to(torch.float8_e4m3fn)


def append(new, cache, scale, slots):
    """One of k and v: new (T, Hk, D), cache (N, P, Hk, D), scale (N, P / block, Hk), on the CPU, in place."""
    N, P, Hk, D = cache.shape
    block = P // scale.shape[1]
    big = torch.finfo(new.dtype).max
    x = new.double()
    x = torch.where(torch.isinf(x), torch.sign(x) * big, x)
    top = CODE_MAX[cache.dtype]
    runs = []
    for i, s in enumerate(slots):
        if not 0 <= s < N * P:
            continue
        if runs and runs[-1][0] == s // block and runs[-1][2] == i:
            runs[-1][2] = i + 1
        else:
            runs.append([s // block, i, i + 1])
    for b, i0, i1 in runs:
        n, j = b * block // P, b * block % P
        first = slots[i0] - b * block
        for h in range(Hk):
            most = torch.nan_to_num(x[i0:i1, h], nan=0.0).abs().max().item()
            s = FLOOR
            if most > top * FLOOR:
                s = 2.0 ** (math.frexp(most)[1] - math.frexp(top)[1])
                s = s if most <= top * s else 2 * s
            if first:
                old = scale[n, j // block, h].item()
                if old >= s:
                    s = old
                else:
                    cache[n, j:j + first, h] = encode(cache[n, j:j + first, h].double() * (old / s), cache.dtype)
            scale[n, j // block, h] = s
            for i in range(i0, i1):
                cache[n, slots[i] - n * P, h] = encode(x[i, h] / s, cache.dtype)


def rows_of(cache, scale, pages, n):
    """Values (n, Hk, D) of keys 0 .. n - 1 in 64 bits and whether their page is in the cache."""
    P, block = cache.shape[1], cache.shape[1] // scale.shape[1]
    j = torch.arange(n)
    page = torch.tensor(pages, dtype=torch.long)[j // P]
    ok = (page >= 0) & (page < cache.shape[0])
    page = page.clamp(0, cache.shape[0] - 1)
    codes = cache.view(torch.uint8)[page, j % P].view(cache.dtype).double()
    return codes * scale[page, j % P // block].double()[..., None], ok


def attend(q, k, v, ok, scale, causal=False, window=(-1, -1), softcap=0.0):
    """One sequence: q (n, H, D), k and v (L, Hk, D) in 64 bits, ok (L,); out (n, H, D), lse (H, n)."""
    n, H, D = q.shape
    L, Hk = k.shape[0], k.shape[1]
    i = torch.arange(n)[:, None] + L - n
    j = torch.arange(L)[None]
    seen = ok[None].expand(n, L).clone()
    if causal:
        window = (window[0], 0)
    if window[0] >= 0:
        seen &= j >= i - window[0]
    if window[1] >= 0:
        seen &= j <= i + window[1]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    lse = torch.full((H, n), math.inf, dtype=torch.float64)
    for h in range(H):
        x = q[:, h].double() @ k[:, h // (H // Hk)].t() * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        for r in range(n):
            s = seen[r]
            if s.any():
                y = x[r, s]
                lse[h, r] = torch.logsumexp(y, 0)
                out[r, h] = torch.exp(y - lse[h, r]) @ v[s, h // (H // Hk)]
    return out, lse
