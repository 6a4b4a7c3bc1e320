"""Rows that the formula makes NaN stay NaN where several workgroups share their keys: the merge must not
take them for rows that see no key (out 0, softmax_lse +inf)."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._quant import Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def call(c, q, **kw):
    return fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32),
                                                page_table=None if c.table is None else c.table.to(DEV), causal=True,
                                                return_softmax_lse=True, **kw)


def check_rows(c, b, out, lse, q, bad, dtype, **how):
    """out (n, H, D), lse (H, n) of sequence b: NaN at the (row, head) pairs of `bad`, as defined elsewhere."""
    for r, h in bad:
        assert out[r, h].isnan().all() and lse[h, r].isnan(), (r, h, out[r, h, :4], lse[h, r])
    keep = torch.ones(q.shape[:2], dtype=torch.bool)
    for r, h in bad:
        keep[r, h] = False
    out, lse = out.cpu(), lse.cpu()
    k, v, ok, top = c.rows(b)
    # the rows left, one at a time where a bad one shares their position
    g = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        if keep[:, h].all():
            check_attend(out[:, h:h + 1], lse[h:h + 1], q[:, h:h + 1], k[:, h // g:h // g + 1], v[:, h // g:h // g + 1], ok, top,
                         dtype, causal=True, **how)
            continue
        for r in range(q.shape[0]):
            if keep[r, h]:
                n = k.shape[0] - (q.shape[0] - 1 - r)  # causal: the keys up to the row's own
                check_attend(out[r:r + 1, h:h + 1], lse[h:h + 1, r:r + 1], q[r:r + 1, h:h + 1], k[:n, h // g:h // g + 1],
                             v[:n, h // g:h // g + 1], ok[:n], top, dtype, causal=True, **how)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq,keys", [(1, 3000), (3, 3000), (1, 20), (2, 20)])
def test_query_rows_in_decode(sq, keys, D, cache, value):
    """Few rows over many keys, which many waves share, and over few, which one holds."""
    print(f"case nan decode {sq} {keys} {D} {cache} {value}", flush=True)
    g = torch.Generator().manual_seed(31)
    c = Cache(g, [keys, 77], 2, D, cache, 64, 32)
    q = torch.randn(2, sq, 4, D, generator=g).to(torch.bfloat16)
    q[0, sq - 1, 1, 5] = value
    out, lse = call(c, q)
    check_rows(c, 0, out[0], lse[0], q[0], [(sq - 1, 1)], torch.bfloat16)
    check_rows(c, 1, out[1], lse[1], q[1], [], torch.bfloat16)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_query_rows_in_cut_items(D, cache, value):
    """Ragged prompts: items that workgroups share."""
    print(f"case nan cut items {D} {cache} {value}", flush=True)
    g = torch.Generator().manual_seed(32)
    rows = [40, 25]
    c = Cache(g, [6000, 1500], 2, D, cache, 64, 32)
    q = torch.randn(sum(rows), 4, D, generator=g).to(torch.float16)
    q[17, 2, 3] = value
    q[39, 0, D - 1] = value
    q[40, 3, 0] = value
    cu = torch.tensor([0, 40, 65], **I32)
    out, lse = call(c, q, cu_seqlens_q=cu, max_seqlen_q=40)
    check_rows(c, 0, out[:40], lse[:, :40], q[:40], [(17, 2), (39, 0)], torch.float16)
    check_rows(c, 1, out[40:], lse[:, 40:], q[40:], [(0, 3)], torch.float16)


@pytest.mark.parametrize("keys", [3000, 50])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq", [1, 60])
def test_only_visible_block_has_a_nan_scale(sq, D, keys):
    """All pages but one are missing, and that one's K scale is NaN: every row is NaN, not empty."""
    print(f"case only nan block {sq} {D} {keys}", flush=True)
    g = torch.Generator().manual_seed(33)
    c = Cache(g, [keys], 2, D, "int8", 16, 16)
    at = 2 if keys == 50 else 61
    page = c.pages[0][at]
    c.table[0, :] = -1
    c.table[0, at] = page
    c.scales[0][page] = math.nan
    q = torch.randn(sq, 4, D, generator=g).to(torch.bfloat16)
    first = max(0, at * 16 - (keys - sq))  # the first row that sees a key of it
    for ragged in (False, True):
        more = dict(cu_seqlens_q=torch.tensor([0, sq], **I32), max_seqlen_q=sq) if ragged else {}
        out, lse = call(c, q if ragged else q[None], **more)
        if not ragged:
            out, lse = out[0], lse[0]
        assert out[first:].isnan().all() and lse[:, first:].isnan().all()
        assert (out[:first] == 0).all() and (lse[:, :first] == math.inf).all()


@pytest.mark.parametrize("sq", [1, 60])
def test_one_block_of_many_has_a_nan_scale(sq):
    """A NaN among finite scores of other workgroups' keys."""
    print(f"case one nan block {sq}", flush=True)
    g = torch.Generator().manual_seed(34)
    c = Cache(g, [3000], 2, 128, "e4m3", 64, 16)
    c.scales[0][c.pages[0][9], 1, 1] = math.nan  # of kv head 1
    q = torch.randn(1, sq, 4, 128, generator=g).to(torch.bfloat16)
    out, lse = call(c, q)
    assert out[0, :, 2:].isnan().all() and lse[0, 2:].isnan().all()
    assert out[0, :, :2].isfinite().all() and lse[0, :2].isfinite().all()
