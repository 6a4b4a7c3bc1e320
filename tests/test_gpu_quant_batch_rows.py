"""Rows of cache_batch_idx that are not in the page table (or the contiguous cache): update_page_table gives such a
request no pages, and attention finds no keys for it, least of all another request's."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._quant import Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("sq", [1, 3, 40])
def test_rows_that_are_not_there(sq, page, ragged):
    print(f"case batch rows {sq} {page} {ragged}", flush=True)
    g = torch.Generator().manual_seed(101)
    c = Cache(g, [256, 100, 199], 2, 64, "int8", page, 32, room=256)
    idx = [2, -1, 0, 3, 2 ** 31 - 1, -2 ** 31, 1]
    lens = [c.lens[i] if 0 <= i < 3 else 150 for i in idx]
    q = torch.randn(len(idx), sq, 8, 64, generator=g).to(torch.bfloat16)
    more = dict(cu_seqlens_q=torch.arange(0, (len(idx) + 1) * sq, sq, **I32), max_seqlen_q=sq) if ragged else {}
    out, lse = fa.flash_attn_with_quantized_kvcache(
        (q.flatten(0, 1) if ragged else q).to(DEV), *c.args(DEV), torch.tensor(lens, **I32), causal=True, return_softmax_lse=True,
        page_table=None if c.table is None else c.table.to(DEV), cache_batch_idx=torch.tensor(idx, **I32), **more)
    if ragged:
        out, lse = out.view(len(idx), sq, 8, 64), lse.view(8, len(idx), sq).transpose(0, 1)
    for b, i in enumerate(idx):
        if 0 <= i < 3:
            check_attend(out[b], lse[b], q[b], *c.rows(i), torch.bfloat16, causal=True)
        else:
            assert (out[b] == 0).all() and (lse[b] == math.inf).all()
