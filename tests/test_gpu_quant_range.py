"""V scales far apart: a row's result depends on the scales of the keys that it sees, weighed by their
probabilities, and on nothing else."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_quant_oracle as qo
from tests._quant import Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def attend(c, q, **kw):
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32),
                                                    page_table=c.table.to(DEV), return_softmax_lse=True, **kw)
    return out.cpu(), lse.cpu()


def v_scales(c, b):
    """Of each key (n, Hk)."""
    j = torch.arange(c.lens[b])
    pages = torch.tensor(c.pages[b])[j // c.page]
    return c.scales[1][pages, j % c.page // c.block].double()


def check(out, lse, q, k, v, ok, t, top, causal, scale=None):
    """out (n, H, D), lse (H, n) of one sequence. The bounds are those of tests/_quant.py's check_attend, but for the
    weights: they are rounded to fp16 in a unit in which the largest p t of the row's own keys is 2^10 at least,
    so off by half a step, 2^-11, or by 2^-35 of that p t, for each of L keys, times the largest code `top`. The exponents
    x + log2 t and their difference from the row's reference are two fp32 sums more: 2^-23 of the largest
    |log2 t| (of 100 at most), relative."""
    n, H, D = q.shape
    L, g = k.shape[0], H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    seen = ok[None].expand(n, L).clone()
    if causal:
        seen &= torch.arange(L)[None] <= torch.arange(n)[:, None] + L - n
    for h in range(H):
        kh, vh, th = k[:, h // g], v[:, h // g], t[:, h // g]
        x = q[:, h].double() @ kh.t() * scale
        big = (q[:, h].double().abs() @ kh.abs().t() * abs(scale))
        x = torch.where(seen, x, -math.inf)
        z = torch.logsumexp(x, -1)
        p = torch.exp(x - z[:, None])
        ref = p @ vh
        size = p @ vh.abs()
        logs = 100 * 2.0 ** -23
        d = (D + 16) * 2.0 ** -24 * torch.where(seen, big, 0.0).amax(1, keepdim=True)
        largest = (p * th.abs()).amax(1, keepdim=True) * top
        eps = torch.finfo(q.dtype).eps / 2
        bound = size * (2.0 ** -11 + 2 * d + (L + 16) * 2.0 ** -24 + logs) + eps * ref.abs() + L * 2.0 ** -34 * largest \
            + torch.finfo(q.dtype).smallest_normal * eps * 2
        got = out[:, h].double()
        assert got.isfinite().all(), f"head {h}: rows {(~got.isfinite().all(1)).nonzero().flatten().tolist()[:9]} are not finite"
        off = ((got - ref).abs() / bound).amax(1)
        assert off.max() <= 1, f"head {h}: row {int(off.argmax())} is off by {off.max():.3g} times its bound"
        bound = d[:, 0] + (L + 16) * 2.0 ** -24 + 2.0 ** -22 * z.abs() + logs
        assert ((lse[h].double() - z).abs() <= bound).all(), f"lse of head {h}"


def whole(c, b, out, lse, q, causal):
    k, v, ok, _ = c.rows(b)
    check(out, lse, q, k, v, ok, v_scales(c, b), qo.CODE_MAX[c.codes[1].dtype], causal)


@pytest.mark.parametrize("exponent", [-98, -99, -110])
@pytest.mark.parametrize("keys", [1024, 1000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_small_scales_to_the_end_of_a_group(D, keys, exponent):
    """1024 keys fill the prefill kernel's groups of blocks to the last."""
    print(f"case small scales {D} {keys} {exponent}", flush=True)
    g = torch.Generator().manual_seed(51)
    c = Cache(g, [keys, 2 * keys], 2, D, "int8", 64, 16)
    c.scales[1].mul_(2.0 ** exponent / 0.03)
    for sq in (1, 40, 230):
        q = torch.randn(2, sq, 4, D, generator=g).to(torch.bfloat16)
        out, lse = attend(c, q)
        for b in range(2):
            whole(c, b, out[b], lse[b], q[b], False)
