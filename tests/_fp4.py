"""4-bit caches for the tests, with everything that no call may read made NaN, and the bounds of the attention's
error over them."""
import math

import torch

from oracle import fa_fp4_oracle as fo
from oracle import fa_quant_oracle as qo

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


class Cache4:
    """A cache on the CPU for sequences of `lens` keys: pages in any order, page 0 unused, rows and table entries that hold
    no key poisoned (scale NaN, an id outside the cache). page 0 (no table): contiguous, `room` rows a sequence."""

    def __init__(self, g, lens, Hk, D, page, room=0, spread=2.0):
        self.page, self.lens = page, list(lens)
        size = page or room
        need = [-(-n // page) for n in lens] if page else [1] * len(lens)
        count = sum(need) + 2 if page else len(lens)
        ids = (torch.randperm(count - 1, generator=g) + 1).tolist() if page else list(range(count))
        self.pages = [[ids.pop(0) for _ in range(n)] for n in need]
        live = torch.zeros(count, size, dtype=torch.bool)
        for pages, n in zip(self.pages, lens):
            for i, p in enumerate(pages):
                live[p, :min(max(n - i * size, 0), size)] = True
        self.codes, self.scales = [], []
        for _ in range(2):
            c = torch.randint(0, 256, (count, size, Hk, D // 2), generator=g, dtype=torch.uint8)
            s = (126 + torch.randn(count, size, Hk, D // 32, generator=g) * spread).round().clamp(1, 254).to(torch.uint8)
            c[~live], s[~live] = 0x77, 255
            self.codes.append(c)
            self.scales.append(s)
        self.table = None
        if page:
            self.table = torch.full((len(lens), max(need) + 1), 0x7fffffff, dtype=torch.int32)
            for r, pages in enumerate(self.pages):
                self.table[r, :len(pages)] = torch.tensor(pages, dtype=torch.int32)

    def args(self, dev):
        """k_cache, v_cache, k_scale, v_scale on the device."""
        return [t.to(dev) for t in (*self.codes, *self.scales)]

    def rows(self, b, dtype):
        """k, v as `dtype` holds them, in 64 bits, and whether their page is in the cache, of sequence b."""
        pages = [b] if self.table is None else self.table[b].tolist()
        k, ok = fo.rows_of(self.codes[0], self.scales[0], pages, self.lens[b])
        v, _ = fo.rows_of(self.codes[1], self.scales[1], pages, self.lens[b])
        return k.to(dtype).double(), v.to(dtype).double(), ok


def check_attend4(out, lse, q, k, v, ok, dtype, scale=None, softcap=0.0, **how):
    """out (n, H, D) and lse (H, n) of one sequence against the definition.

    The bounds count: q and the values of K and V are 16-bit operands, whose products are exact; a score is an fp32 sum of D
    of them and a handful of roundings, so off by less than d = (D + 16) 2^-24 X, X the sum of the products' sizes (a
    soft cap adds the 2^-21 of its tanh, times the cap); e^x moves by d, sums of n of them by n 2^-24; the weights are
    rounded to dtype before they meet V: half a step, or where fp16 has no more exponents 2^-25 of their unit, which is at
    most 2^-10 of the largest's (so 2^-34 for each of L keys and the largest |v|, the sum of the weights being at least
    1); the result is rounded once more."""
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
    top = v.nan_to_num(0.0).abs().max().item() if L else 0.0
    bound = size * (half + 2 * d + (L + 16) * 2.0 ** -24) + half * ref.abs() + torch.finfo(dtype).smallest_normal * half * 2
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
