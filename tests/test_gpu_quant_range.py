"""V scales far apart: a row's result depends on the scales of the keys that it sees, weighed by their
probabilities, and on nothing else."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_quant_oracle as qo
from tests._quant import Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
# query rows, heads (2 key / value heads): few rows, and many in a call of one and of two 32-row blocks a wave
SHAPES = [(1, 4), (4, 4), (12, 4), (40, 4), (230, 4)]


def attend(c, q, **kw):
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32),
                                                    page_table=c.table.to(DEV), return_softmax_lse=True, **kw)
    return out.cpu(), lse.cpu()


def v_scales(c, b):
    """Of each key (n, Hk)."""
    j = torch.arange(c.lens[b])
    pages = torch.tensor(c.pages[b], dtype=torch.long)[j // c.page]
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


@pytest.mark.parametrize("exponent", [30, 60, 100])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq,H", SHAPES)
def test_large_scale_of_a_hidden_block(sq, H, D, cache, exponent):
    """Causal: the last block of 16 keys, which the first rows do not see."""
    print(f"case hidden large {sq} {H} {D} {cache} {exponent}", flush=True)
    g = torch.Generator().manual_seed(52)
    sk = 1389  # ends 13 keys into a block
    c = Cache(g, [sk], 2, D, cache, 64, 16)
    last = sk - 1
    c.scales[1][c.pages[0][last // 64], last % 64 // 16] = 2.0 ** exponent
    q = torch.randn(1, sq, H, D, generator=g).to(torch.bfloat16)
    out, lse = attend(c, q, causal=True)
    whole(c, 0, out[0], lse[0], q[0], True)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq,H", SHAPES)
def test_large_scales_left_of_a_window(sq, H, D):
    """The first rows see blocks of a large scale that the window hides from the last ones."""
    print(f"case window large {sq} {H} {D}", flush=True)
    g = torch.Generator().manual_seed(53)
    sk, left = 700, 290
    c = Cache(g, [sk], 2, D, "int8", 64, 16)
    first = max(sk - sq - left, 0)  # the first key that any row sees
    c.scales[1][c.pages[0][first // 64], first % 64 // 16] = 2.0 ** 70
    q = torch.randn(1, sq, H, D, generator=g).to(torch.bfloat16)
    out, lse = attend(c, q, causal=True, window_size=(left, 0))
    k, v, ok, _ = c.rows(0)
    for r in range(0, sq, max(1, sq // 9)):
        i = sk - sq + r
        lo = max(i - left, 0)
        check(out[0, r:r + 1], lse[0, :, r:r + 1], q[0, r:r + 1], k[lo:i + 1], v[lo:i + 1], ok[lo:i + 1], v_scales(c, 0)[lo:i + 1],
              127.0, False)


@pytest.mark.parametrize("push", [-150.0, 150.0])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq,H", SHAPES)
def test_large_scale_of_an_unlikely_block(sq, H, D, push):
    """A block of scale 2^90 whose scores lie 150 below the others' (push < 0), or before one whose scores lie 150
    above all others: its p is 0 in 32 bits, and so is what it adds."""
    print(f"case unlikely large {sq} {H} {D} {push}", flush=True)
    g = torch.Generator().manual_seed(54)
    sk = 1300
    c = Cache(g, [sk], 2, D, "int8", 64, 16)
    q = torch.randn(1, sq, H, D, generator=g)
    q[..., 0] = 8.0
    c.codes[0][..., 0] = 0
    large, pushed = (10, 10) if push < 0 else (10, 31)  # blocks of 16 keys
    at = lambda i: (c.pages[0][i // 4], i % 4)  # noqa: E731
    c.scales[1][at(large)] = 2.0 ** 90
    page, i = at(pushed)
    c.codes[0][page, 16 * i:16 * i + 16] = 0
    c.codes[0][page, 16 * i:16 * i + 16, :, 0] = 127 if push > 0 else -127
    c.scales[0][page, i] = abs(push) / (8 * 127 * D ** -0.5)
    q = q.to(torch.bfloat16)
    out, lse = attend(c, q, causal=True)
    whole(c, 0, out[0], lse[0], q[0], True)


@pytest.mark.parametrize("how", ["far", "near", "zero", "first"])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq,H", SHAPES)
def test_scales_of_every_size(sq, H, D, cache, how):
    """Each block another scale: within 2^+-70, within 2^+-30, one in four 0, the first 200 keys tiny."""
    print(f"case every size {sq} {H} {D} {cache} {how}", flush=True)
    g = torch.Generator().manual_seed(55)
    c = Cache(g, [2100, 130], 2, D, cache, 64, 16)
    s = c.scales[1]
    if how == "zero":
        s.mul_((torch.rand(s.shape, generator=g) > 0.25).float())
    elif how == "first":
        for page in c.pages[0][:3]:
            s[page] = 2.0 ** -100
    else:
        r = 70 if how == "far" else 30
        s.copy_(2.0 ** (torch.rand(s.shape, generator=g) * 2 * r - r))
    q = torch.randn(2, sq, H, D, generator=g).to(torch.bfloat16)
    out, lse = attend(c, q, causal=True)
    for b in range(2):
        n = max(0, sq - c.lens[b])  # rows that see no key
        assert (out[b, :n] == 0).all() and (lse[b, :, :n] == math.inf).all()
        whole(c, b, out[b, n:], lse[b, :, n:], q[b, n:], True)


@pytest.mark.parametrize("cache", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("sq", [8, 60])
def test_appended_infinity(sq, cache):
    """A value row with an infinity, as the append stores it, stays with the rows that see it."""
    print(f"case appended infinity {sq} {cache}", flush=True)
    g = torch.Generator().manual_seed(56)
    sk, D = 500, 64
    k, v = (torch.randn(sk, 2, D, generator=g).to(torch.bfloat16) for _ in range(2))
    v[498, :, 7] = math.inf
    kc, vc = (torch.zeros(9, 64, 2, D).to(cache).to(DEV) for _ in range(2))
    ks, vs = (torch.zeros(9, 4, 2, device=DEV) for _ in range(2))
    slots = torch.arange(64, 64 + sk, device=DEV)
    fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), kc, vc, ks, vs, slots)
    q = torch.randn(1, sq, 4, D, generator=g).to(torch.bfloat16)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), kc, vc, ks, vs, torch.tensor([sk], **I32),
                                                    page_table=torch.arange(1, 9, **I32)[None], causal=True, return_softmax_lse=True)
    n = sq - (sk - 496)  # the queries that see no key of the last block
    codes = lambda x, s: (qo.rows_of(x.cpu(), s.cpu(), list(range(1, 9)), 496))  # noqa: E731
    (kk, ok), (vv, _) = codes(kc, ks), codes(vc, vs)
    top = vs.cpu().view(-1, 2)[4:4 + 31].max().item() * qo.CODE_MAX[cache]
    check_attend(out[0, :n], lse[0, :, :n], q[0, :n], kk, vv, ok, top, torch.bfloat16, causal=True)
