"""Scales that are no numbers at keys that some rows of a call do not see: those rows
keep their results, the others are NaN or infinite as the formula says."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._quant import TYPES, Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("what", [(0, math.nan), (1, math.nan), (1, math.inf), (1, -math.inf)])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("sq,H,D", [(24, 2, 64), (24, 2, 128), (24, 2, 256), (90, 4, 64), (90, 4, 128), (150, 8, 128), (90, 4, 256)])
def test_scales_of_hidden_blocks(sq, H, D, cache, what):
    """Causal: the last block of 16 keys, with such a scale, is seen by the last queries only."""
    print(f"case hidden {sq} {H} {D} {cache} {what}", flush=True)
    g = torch.Generator().manual_seed(21)
    sk = 413
    c = Cache(g, [sk], 2, D, cache, 64, 16)
    last = sk - 1
    page = c.pages[0][last // 64]
    seen = sk - last % 16 - 1  # keys before the block
    k, v, ok, top = c.rows(0)
    c.scales[what[0]][page, last % 64 // 16] = what[1]
    q = torch.randn(1, sq, H, D, generator=g).to(torch.bfloat16)
    out, lse = fa.flash_attn_with_quantized_kvcache(
        q.to(DEV), *c.args(DEV), torch.tensor([sk], dtype=torch.int32, device=DEV), page_table=c.table.to(DEV), causal=True,
        return_softmax_lse=True)
    n = sq - (sk - seen)  # the queries that do not see it
    check_attend(out[0, :n], lse[0, :, :n], q[0, :n], k[:seen], v[:seen], ok[:seen], top, torch.bfloat16, causal=True)
    assert not out[0, n:].isfinite().all(-1).any()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("Hk,lens", [(2, [700, 3, 40, 0, 129, 1, 260]), (8, [300, 300, 300]), (1, [1100])])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cut_items(D, Hk, lens, dt):
    """Ragged batches whose items the workgroups share, over several groups of 1024 keys."""
    print(f"case cut {D} {Hk} {lens} {dt}", flush=True)
    g = torch.Generator().manual_seed(22)
    keys = [n + (1900 if i % 3 == 0 else 5) for i, n in enumerate(lens)]
    c = Cache(g, keys, Hk, D, "int8", 32, 16)
    q = torch.randn(sum(lens), 2 * Hk, D, generator=g).to(TYPES[dt])
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    out, lse = fa.flash_attn_with_quantized_kvcache(
        q.to(DEV), *c.args(DEV), torch.tensor(keys, dtype=torch.int32, device=DEV), page_table=c.table.to(DEV),
        cu_seqlens_q=cu.to(DEV), max_seqlen_q=max(lens), causal=True, return_softmax_lse=True)
    for b, n in enumerate(lens):
        if n:
            r = slice(int(cu[b]), int(cu[b + 1]))
            check_attend(out[r], lse[:, r], q[r], *c.rows(b), TYPES[dt], causal=True)
