"""Sizes and windows that do not fit in the 32 bits of the C entries are refused, or taken for what they mean."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._quant import Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("left", [-2 ** 33, -2 ** 32 + 3, -2 ** 31 - 1, 2 ** 40])
@pytest.mark.parametrize("right", [-2 ** 33, 2 ** 35 + 2])
def test_windows(left, right):
    print(f"case windows {left} {right}", flush=True)
    g = torch.Generator().manual_seed(131)
    c = Cache(g, [300], 2, 64, "int8", 64, 16)
    q = torch.randn(1, 20, 4, 64, generator=g).to(torch.bfloat16)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor([300], **I32), page_table=c.table.to(DEV),
                                                    window_size=(left, right), return_softmax_lse=True)
    check_attend(out[0], lse[0], q[0], *c.rows(0), torch.bfloat16)


@pytest.mark.parametrize("pages", [2 ** 31, 2 ** 32 + 6])
def test_pages(pages):
    """Views of one page, no memory behind the others."""
    print(f"case pages {pages}", flush=True)
    kc = torch.zeros(1, 16, 1, 16, dtype=torch.int8, device=DEV).expand(pages, 16, 1, 16)
    s = torch.ones(1, 1, 1, device=DEV).expand(pages, 1, 1)
    q = torch.zeros(1, 1, 1, 16, dtype=torch.float16, device=DEV)
    one = torch.ones(1, **I32)
    with pytest.raises(RuntimeError, match="number of pages must be less than 2\\^31"):
        fa.flash_attn_with_quantized_kvcache(q, kc, kc, s, s, one, page_table=one[:, None])
    with pytest.raises(RuntimeError, match="number of pages must be less than 2\\^31"):
        fa.append_quantized_kvcache(q[0], q[0], kc, kc, s, s, torch.full((1,), -1, device=DEV))


def test_heads():
    print("case heads", flush=True)
    n = 2 ** 32 + 1
    kc = torch.zeros(1, 16, 1, 16, dtype=torch.int8, device=DEV).expand(1, 16, n, 16)
    s = torch.ones(1, 1, 1, device=DEV).expand(1, 1, n)
    q = torch.zeros(1, 1, 1, 16, dtype=torch.float16, device=DEV)
    one = torch.ones(1, **I32)
    with pytest.raises(RuntimeError, match="heads must be less than 2\\^31"):
        fa.flash_attn_with_quantized_kvcache(q, kc, kc, s, s, one)
