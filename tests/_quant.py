"""Quantised caches for the tests, with everything that no call may read made NaN
(or the largest code), and the bounds of the attention's error."""
import math

import torch

from oracle import fa_quant_oracle as qo

E4M3 = torch.float8_e4m3fn
CACHES = {"int8": torch.int8, "e4m3": E4M3}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


class Cache:
    """A cache on the CPU for sequences of `lens` keys: pages in any order, page 0 unused, rows, scales
    and table entries that hold no key poisoned. page 0 (no table): contiguous, `room` rows a sequence."""

    def __init__(self, g, lens, Hk, D, cache, page, block, room=0, spread=0.3):
        dt = CACHES[cache]
        self.page, self.block, self.lens = page, block, list(lens)
        size = page or room
        need = [-(-n // page) for n in lens] if page else [1] * len(lens)
        count = sum(need) + 2 if page else len(lens)
        ids = (torch.randperm(count - 1, generator=g) + 1).tolist() if page else list(range(count))
        self.pages = [[ids.pop(0) for _ in range(n)] for n in need]
        live = torch.zeros(count, size, dtype=torch.bool)
        for pages, n in zip(self.pages, lens):
            for i, p in enumerate(pages):
                live[p, :min(max(n - i * size, 0), size)] = True
        self.scales = []
        self.codes = []
        for _ in range(2):
            top = qo.CODE_MAX[dt]
            x = torch.randn(count, size, Hk, D, generator=g).mul_(top / 3.5).clamp_(-top, top)
            c = x.round().to(dt) if cache == "int8" else x.to(dt)
            c.view(torch.uint8)[~live] = 0x7f
            s = torch.exp(torch.randn(count, size // block, Hk, generator=g) * spread) * (3.5 / top)
            s[~live.view(count, size // block, block).any(-1)] = math.nan
            self.codes.append(c)
            self.scales.append(s)
        if page:
            wide = max(need) + 1
            self.table = torch.full((len(lens), wide), 0x7fffffff, dtype=torch.int32)
            for r, pages in enumerate(self.pages):
                self.table[r, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        else:
            self.table = None

    def args(self, dev):
        """k_cache, v_cache, k_scale, v_scale on the device."""
        return [t.to(dev) for t in (*self.codes, *self.scales)]

    def rows(self, b):
        """k, v in 64 bits, whether their page is in the cache, and the largest value that its v could hold, of
        sequence b."""
        n = self.lens[b]
        if self.table is None:
            pages = [b]
        else:
            pages = self.table[b].tolist()
        k, ok = qo.rows_of(self.codes[0], self.scales[0], pages, n)
        v, _ = qo.rows_of(self.codes[1], self.scales[1], pages, n)
        return k, v, ok, largest(self.codes[1], self.scales[1])


def largest(codes, scale):
    return scale.nan_to_num(0.0).abs().max().item() * qo.CODE_MAX[codes.dtype]


def check_attend(out, lse, q, k, v, ok, top, dtype, scale=None, softcap=0.0, **how):
    """out (n, H, D) and lse (H, n) of one sequence against the definition.

    The bounds count: the 16-bit codes of q, K and V enter their products exactly;
    a score is an fp32 sum of D products and a handful of roundings, so off by
    less than d = (D + 16) 2^-24 X, X the sum of the products' sizes (a soft cap
    adds the 2^-21 of its tanh, times the cap); e^x moves by d, sums of n of them
    by n 2^-24; the weights p t of the V scales t are rounded to fp16 before they
    meet V: half a step, 2^-11, or 2^-25 of the unit they are kept in, which is at
    most 2 max t 2^-14 in the decode kernel and 2 max t 2^-10 in the other, whose lazy
    maximum needs the room (the sum of p is at least 1 in both), so 2^-34 max t for
    each of L keys and `top`, max t times the largest code, for what they multiply;
    the result is rounded once more."""
    n, H, D = q.shape
    L, g = k.shape[0], H // k.shape[1]
    if scale is None:
        scale = D ** -0.5
    ref, ref_lse = qo.attend(q, k, v, ok, scale, softcap=softcap, **how)
    size, _ = qo.attend(q, k, v.abs(), ok, scale, softcap=softcap, **how)  # sum of p |v|
    x = torch.zeros(n, H, 1, dtype=torch.float64)
    if L:
        for h in range(H):
            x[:, h, 0] = (q[:, h].double().abs() @ k[:, h // g].abs().t()).nan_to_num(0.0).amax(1) * abs(scale)
    d = (D + 16) * 2.0 ** -24 * x + (2.0 ** -21 * softcap)
    got = out.detach().cpu().double()
    assert not torch.isnan(got).any(), "NaN in out"
    half = torch.finfo(dtype).eps / 2
    bound = size * (2.0 ** -11 + 2 * d + (L + 16) * 2.0 ** -24) + half * ref.abs() + torch.finfo(dtype).smallest_normal * half * 2
    bound = bound + L * 2.0 ** -34 * top
    worst = ((got - ref).abs() / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1, f"out {worst:.2f} times its bound"
    got = lse.detach().cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(ref_lse)) and not (got == -math.inf).any()
    fin = ~torch.isinf(ref_lse)
    bound = d[..., 0].t() + (L + 16) * 2.0 ** -24 + 2.0 ** -22 * ref_lse.abs()
    bad = ((got - ref_lse).abs()[fin] / bound[fin]).max().item() if fin.any() else 0.0
    assert bad <= 1, f"lse {bad:.2f} times its bound"
    return worst
