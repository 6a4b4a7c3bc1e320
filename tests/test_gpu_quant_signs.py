"""Scales below 0, subnormal ones and code -128, which no append writes but a cache may hold; softmax scales of either sign."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._quant import Cache
from tests.test_gpu_quant_range import check, v_scales

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def attend(c, q, **kw):
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32),
                                                    page_table=c.table.to(DEV), causal=True, return_softmax_lse=True, **kw)
    return out.cpu(), lse.cpu()


def whole(c, out, lse, q, **kw):
    for b in range(len(c.lens)):
        k, v, ok, _ = c.rows(b)
        n = max(0, q.shape[1] - c.lens[b])
        assert (out[b, :n] == 0).all() and (lse[b, :, :n] == math.inf).all()
        check(out[b, n:], lse[b, :, n:], q[b, n:], k, v, ok, v_scales(c, b), 128.0 if c.codes[1].dtype == torch.int8 else 448.0, True, **kw)


@pytest.mark.parametrize("which", [(0,), (1,), (0, 1)])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("sq,D", [(1, 64), (3, 128), (7, 80), (40, 64), (40, 192), (230, 128)])
def test_negative_scales(sq, D, cache, which):
    print(f"case negative scales {sq} {D} {cache} {which}", flush=True)
    g = torch.Generator().manual_seed(141)
    c = Cache(g, [1300, 77], 2, D, cache, 64, 16)
    for i in which:
        c.scales[i].mul_(1 - 2 * torch.randint(0, 2, c.scales[i].shape, generator=g))
    q = torch.randn(2, sq, 4, D, generator=g).to(torch.bfloat16)
    for scale in (None, -0.2):
        out, lse = attend(c, q, softmax_scale=scale)
        whole(c, out, lse, q, scale=scale)


@pytest.mark.parametrize("low", [-149, -132, -128])
@pytest.mark.parametrize("sq", [1, 5, 60])
def test_subnormal_scales(sq, low):
    """Of V, some of them or all; of K, where a large softmax scale makes up for it."""
    print(f"case subnormal scales {sq} {low}", flush=True)
    g = torch.Generator().manual_seed(142)
    for part in (0.3, 1.0):
        c = Cache(g, [300, 40], 2, 64, "int8", 64, 16)
        tiny = torch.rand(c.scales[1].shape, generator=g) < part
        c.scales[1][tiny] = 2.0 ** low * 3
        q = torch.randn(2, sq, 4, 64, generator=g).to(torch.bfloat16)
        out, lse = attend(c, q)
        whole(c, out, lse, q)


@pytest.mark.parametrize("sq", [1, 5, 60])
def test_lowest_code(sq):
    print(f"case lowest code {sq}", flush=True)
    g = torch.Generator().manual_seed(143)
    c = Cache(g, [300, 40], 2, 64, "int8", 64, 16)
    for x in c.codes:
        x[torch.rand(x.shape, generator=g) < 0.2] = -128
    q = torch.randn(2, sq, 4, 64, generator=g).to(torch.float16)
    out, lse = attend(c, q)
    whole(c, out, lse, q)
