"""The 4-bit cache from its definition, in Python and 64 bits on the CPU: codes and
scales of new rows, and the values that a cache holds. Test infrastructure, written for
reading: a group of 32 channels at a time is enough to follow."""
import math

import torch

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # by code; the upper half are the negatives
LOWEST = -100
HIGHEST = {torch.float16: 13, torch.bfloat16: 125}


def group(x, dtype):
    """(codes, scale byte) of 32 values, a list of floats that came in `dtype`."""
    if any(math.isnan(v) for v in x):
        big = torch.finfo(dtype).max
        byte = 255
    else:
        big, byte = torch.finfo(dtype).max, None
    x = [math.copysign(big, v) if math.isinf(v) or math.isnan(v) else v for v in x]
    most = max(abs(v) for v in x)
    e = LOWEST
    while most > 6.0 * 2.0 ** e and e < HIGHEST[dtype]:
        e += 1
    codes = []
    for v in x:
        a = abs(v) / 2.0 ** e
        # the nearest; of two that are equally near, the even code
        c = min(range(8), key=lambda i: (abs(a - GRID[i]), i % 2))
        codes.append(c + (8 if math.copysign(1.0, v) < 0 else 0))
    return codes, e + 127 if byte is None else byte


def append(new, cache, scale, slots):
    """One of k and v: new (T, Hk, D), cache (N, P, Hk, D / 2) and scale (N, P, Hk, D / 32) uint8, on the CPU, in place.
    The codes of a group with the scale NaN say nothing."""
    N, P, Hk, half = cache.shape
    for i, s in enumerate(slots):
        if not 0 <= s < N * P:
            continue
        for h in range(Hk):
            for g in range(half // 16):
                codes, byte = group(new[i, h, 32 * g:32 * g + 32].double().tolist(), new.dtype)
                pairs = [a + 16 * b for a, b in zip(codes[0::2], codes[1::2])]
                cache[s // P, s % P, h, 16 * g:16 * g + 16] = torch.tensor(pairs, dtype=torch.uint8)
                scale[s // P, s % P, h, g] = byte


def values(codes, scale):
    """Rows of codes (..., D / 2) and scale bytes (..., D / 32) in 64 bits."""
    known = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64)
    x = known[torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()]
    s = torch.where(scale == 255, math.nan, 2.0 ** (scale.double() - 127.0))
    return x * s.repeat_interleave(32, -1)


def rows_of(cache, scale, pages, n):
    """Values (n, Hk, D) of keys 0 .. n - 1 in 64 bits and whether their page is in the cache."""
    P = cache.shape[1]
    j = torch.arange(n)
    page = torch.tensor(pages, dtype=torch.long)[j // P]
    ok = (page >= 0) & (page < cache.shape[0])
    page = page.clamp(0, cache.shape[0] - 1)
    return values(cache[page, j % P], scale[page, j % P]), ok
