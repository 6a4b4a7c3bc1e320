"""The 4-bit decode kernel where values of V leave the range that fp16 holds exactly, amid a wave's tiles, and where
groups of V hold zeros under any scale."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._fp4 import Cache4, check_attend4

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def run(c, q, **kw):
    return fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32), page_table=c.table.to(DEV),
                                                return_softmax_lse=True, **kw)


def check(c, q, out, lse):
    for b in range(len(c.lens)):
        check_attend4(out[b], lse[b], q[b], *c.rows(b, torch.bfloat16), torch.bfloat16)


# One sequence of up to 191 keys is one wave's (a wave has two tiles of 64 keys at least); of 4 heads each has its wave.
@pytest.mark.parametrize("lens", [[128], [190], [191, 150, 128]])
@pytest.mark.parametrize("D,H,Hk", [(64, 4, 1), (128, 8, 4), (256, 4, 1), (64, 32, 1), (64, 20, 1)])
@pytest.mark.parametrize("byte", [90, 103, 141, 150])
def test_scales_out_of_range_after_ordinary_ones(byte, D, H, Hk, lens):
    """Ordinary values in the first tile and in most of the others; one key of the second tile, and none or one of the third,
    has one group of 32 channels out of the range, so that the other channels and the lse show what became of the sums
    before. Up to 16 query heads of a kv head are one row tile, 20 and 32 two."""
    print(f"case fp4 wide {byte} {D} {H} {Hk} {lens}", flush=True)
    g = torch.Generator().manual_seed(31)
    c = Cache4(g, lens, Hk, D, 16)
    for b in range(len(lens)):
        for key in (100, 140):
            if key < lens[b]:
                c.scales[1][c.pages[b][key // 16], key % 16, :, D // 32 - 1] = byte
                c.codes[1][c.pages[b][key // 16], key % 16, :, -16:] = 0x75  # 3 and 6
    q = torch.randn(len(lens), 1, H, D, generator=g).to(torch.bfloat16)
    out, lse = run(c, q)
    check(c, q, out, lse)


@pytest.mark.parametrize("D,H,Hk", [(64, 4, 1), (128, 8, 4), (256, 4, 1), (64, 32, 1), (128, 32, 1)])
@pytest.mark.parametrize("dead", ["some", "all"])
def test_groups_of_zeros(dead, D, H, Hk):
    """Groups whose codes are 0 or -0 hold zeros under any scale: the byte that the append gives them, that of a cleared
    cache, the largest. One group of small values that are not zeros among them."""
    print(f"case fp4 zero groups {dead} {D} {H} {Hk}", flush=True)
    g = torch.Generator().manual_seed(32)
    lens = [191, 700, 64, 1]
    c = Cache4(g, lens, Hk, D, 16)
    codes, scales = c.codes[1], c.scales[1]
    zero = torch.rand(scales.shape, generator=g) < (0.4 if dead == "some" else 2.0)
    bytes_ = torch.tensor([0, 27, 27, 254], dtype=torch.uint8)[torch.randint(0, 4, scales.shape, generator=g)]
    live = scales != 255
    scales.copy_(torch.where(zero & live, bytes_, scales))
    signs = torch.randint(0, 2, codes.shape, generator=g, dtype=torch.uint8) * 0x80 + torch.randint(0, 2, codes.shape, generator=g, dtype=torch.uint8) * 8
    codes.copy_(torch.where((zero & live).repeat_interleave(16, -1), signs, codes))
    q = torch.randn(len(lens), 1, H, D, generator=g).to(torch.bfloat16)
    out, lse = run(c, q)
    check(c, q, out, lse)
    at = c.pages[1][300 // 16], 300 % 16
    scales[at] = 60
    codes[at] = 0x31
    out, lse = run(c, q)
    check(c, q, out, lse)
