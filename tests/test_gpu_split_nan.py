"""Rows that the formula makes NaN in calls whose keys several workgroups share (split-KV): out and softmax_lse are
NaN as in calls that are not split, never those of the other splits or of a row that sees no key."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def plain(q, k, v):
    """Out (n, H, D) and lse (H, n) of one sequence in 64 bits, no mask."""
    g = q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(g, 1).transpose(0, 1) for x in (k, v))
    x = q.double().transpose(0, 1) @ k.transpose(1, 2) * q.shape[-1] ** -0.5
    return (torch.softmax(x, -1) @ v).transpose(0, 1), torch.logsumexp(x, -1)


def check(out, lse, q, k, v, bad):
    """`bad` (n, H): the rows that are NaN; the others within what 16-bit weights and results leave."""
    out, lse = out.cpu().double(), lse.cpu().double()
    q, k, v = q.double(), k.double(), v.double()
    assert out[bad].isnan().all(), out[bad].flatten()[:8]
    assert lse[bad.t()].isnan().all(), lse[bad.t()].flatten()[:8]
    ref, ref_lse = plain(q.nan_to_num(0), k.nan_to_num(0), v)
    # weights that sum to 1 and the result are rounded by 2^-9 (bf16) of |v| < 6 at most, twice that for the
    # exponentials' and sums' own errors; lse: fp32 products of 256 terms, |score| < 2^6
    assert ((out - ref)[~bad].abs() <= 6 * 2.0 ** -7).all()
    assert ((lse - ref_lse)[~bad.t()].abs() <= 2.0 ** -9).all()


@pytest.mark.parametrize("what", ["q", "k"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sq,keys", [(1, 8000), (2, 8000), (1, 30), (48, 8000), (48, 100), (200, 4000)])
def test_kvcache(sq, keys, D, what):
    print(f"case split nan kvcache {sq} {keys} {D} {what}", flush=True)
    g = torch.Generator().manual_seed(41)
    q, k, v = (torch.randn(s, generator=g).to(torch.bfloat16) for s in ((1, sq, 4, D), (1, keys, 2, D), (1, keys, 2, D)))
    bad = torch.zeros(sq, 4, dtype=torch.bool)
    if what == "q":
        q[0, sq - 1, 1, 3] = math.nan
        bad[sq - 1, 1] = True
    else:
        k[0, keys // 3, 1, 3] = math.nan  # every row of the heads 2 and 3 sees it
        bad[:, 2:] = True
    out, lse = fa.flash_attn_with_kvcache(q.to(DEV), k.to(DEV), v.to(DEV), cache_seqlens=keys, return_softmax_lse=True)[:2]
    if what == "k":
        k[0, keys // 3, 1, 3] = 0
    check(out[0], lse[0], q[0], k[0], v[0], bad)


@pytest.mark.parametrize("num_splits", [1, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_dense(D, num_splits, softcap):
    print(f"case split nan dense {D} {num_splits} {softcap}", flush=True)
    g = torch.Generator().manual_seed(42)
    q, k, v = (torch.randn(s, generator=g).to(torch.float16) for s in ((1, 130, 2, D), (1, 3000, 2, D), (1, 3000, 2, D)))
    q[0, 7, 1, 0] = math.nan
    q[0, 129, 0, D - 1] = math.nan
    bad = torch.zeros(130, 2, dtype=torch.bool)
    bad[7, 1] = bad[129, 0] = True
    out, lse = ops.fwd(q.to(DEV), k.to(DEV), v.to(DEV), None, 0.0, D ** -0.5, False, -1, -1, softcap, num_splits=num_splits)
    out, lse = out[0].cpu(), lse[0].cpu()
    if softcap:
        assert out[bad].isnan().all() and lse[bad.t()].isnan().all()
        assert out[~bad].isfinite().all() and lse[~bad.t()].isfinite().all()
    else:
        check(out, lse, q[0], k[0], v[0], bad)


@pytest.mark.parametrize("sq", [1, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_fp8(D, sq):
    """The only NaN of e4m3 in one q row."""
    print(f"case split nan fp8 {sq} {D}", flush=True)
    g = torch.Generator().manual_seed(43)
    q, k, v = (torch.randn(s, generator=g) for s in ((1, sq, 4, D), (1, 6000, 2, D), (1, 6000, 2, D)))
    q[0, 0, 2, 1] = math.nan
    one = torch.ones(1, 2, device=DEV)
    out, lse = fa.flash_attn_with_kvcache(q.to(E4M3).to(DEV), k.to(E4M3).to(DEV), v.to(E4M3).to(DEV), cache_seqlens=6000,
                                          q_descale=one, k_descale=one, v_descale=one, return_softmax_lse=True)[:2]
    bad = torch.zeros(sq, 4, dtype=torch.bool)
    bad[0, 2] = True
    out, lse = out[0].cpu(), lse[0].cpu()
    assert out[bad].isnan().all() and lse[bad.t()].isnan().all()
    assert out[~bad].isfinite().all() and lse[~bad.t()].isfinite().all()


def test_ragged_batch():
    """Decoding rows and prompt rows in one call; a sequence without keys keeps out 0 and lse +inf."""
    print("case split nan ragged", flush=True)
    g = torch.Generator().manual_seed(44)
    rows, keys = [1, 60, 3, 1], [5000, 3000, 700, 0]
    q = torch.randn(sum(rows), 8, 128, generator=g).to(torch.bfloat16)
    kc, vc = (torch.randn(4, 5000, 2, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    at = [0, 1, 61, 64, 65]
    for b, r in ((0, 0), (1, 33), (2, 2)):
        q[at[b] + r, 5, 9] = math.nan
    cu = torch.tensor(at, dtype=torch.int32, device=DEV)
    # a contiguous cache by pages of its own: the page table of one page a sequence
    table = torch.arange(4, dtype=torch.int32, device=DEV)[:, None]
    out, lse = fa.flash_attn_with_kvcache(q.to(DEV), kc[:, :4992].contiguous().to(DEV), vc[:, :4992].contiguous().to(DEV),
                                          cache_seqlens=torch.tensor([4992, 3000, 700, 0], dtype=torch.int32, device=DEV),
                                          page_table=table, cu_seqlens_q=cu, max_seqlen_q=60, return_softmax_lse=True)[:2]
    for b, r in ((0, 0), (1, 33), (2, 2)):
        n = min(keys[b], 4992)
        bad = torch.zeros(rows[b], 8, dtype=torch.bool)
        bad[r, 5] = True
        s = slice(at[b], at[b + 1])
        check(out[s], lse[:, s], q[s], kc[b, :n], vc[b, :n], bad)
    assert (out[64] == 0).all() and (lse[:, 64] == math.inf).all()
