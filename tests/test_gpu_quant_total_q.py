"""cu_seqlens_q that goes past the rows of q: nothing past them is read or written, and the rows that are there
keep their positions."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import capi
from tests._quant import Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,total", [([3, 5, 2], 6), ([2, 2, 2], 2), ([40, 60, 3], 77), ([1, 90, 0, 1], 91), ([300, 20], 299)])
def test_rows_past_the_end(rows, total, causal):
    """The C entry, on buffers that go on behind total_q."""
    print(f"case rows past the end {rows} {total} {causal}", flush=True)
    g = torch.Generator().manual_seed(61)
    have = [700, 20, 31, 5][:len(rows)]
    left = [max(0, min(sum(rows[:i + 1]), total) - min(sum(rows[:i]), total)) for i in range(len(rows))]
    c = Cache(g, [h + n for h, n in zip(have, left)], 2, 64, "int8", 64, 16)  # keys of dropped tokens: poisoned or no page
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **I32)
    more = sum(rows)
    q = torch.full((more, 4, 64), float("nan"), dtype=torch.bfloat16)
    q[:total] = torch.randn(total, 4, 64, generator=g).to(torch.bfloat16)
    qd = q.to(DEV)
    out, lse = torch.full_like(qd, 7.0), torch.full((4 * total + more,), 7.0, device=DEV)
    k, v, ks, vs = c.args(DEV)
    table = torch.nn.functional.pad(c.table, (0, 6), value=0x7fffffff).to(DEV)
    lens = torch.tensor([h + n for h, n in zip(have, rows)], **I32)
    cache = 2 * 64
    p = capi.new_quant_fwd_params(
        dtype=capi.FA_DTYPE_BF16, cache_dtype=capi.FA_DTYPE_INT8, batch=len(rows), seqlen_q=max(rows), nheads=4, nheads_k=2,
        headdim=64, num_pages=k.shape[0], page_size=64, scale_block=16, q=qd.data_ptr(), q_row_stride=256, q_head_stride=64,
        k=k.data_ptr(), k_page_stride=64 * cache, k_row_stride=cache, k_head_stride=64,
        v=v.data_ptr(), v_page_stride=64 * cache, v_row_stride=cache, v_head_stride=64,
        k_scale=ks.data_ptr(), k_scale_page_stride=8, k_scale_block_stride=2, k_scale_head_stride=1,
        v_scale=vs.data_ptr(), v_scale_page_stride=8, v_scale_block_stride=2, v_scale_head_stride=1,
        out=out.data_ptr(), out_row_stride=256, out_head_stride=64, softmax_lse=lse.data_ptr(),
        cache_seqlens=lens.data_ptr(), cu_seqlens_q=cu.data_ptr(), total_q=total, page_table=table.data_ptr(),
        page_table_row_stride=table.shape[1], table_rows=len(rows), max_pages=table.shape[1], softmax_scale=0.125,
        is_causal=int(causal))
    st, n = capi.quant_fwd_workspace_size(p)
    assert st == capi.FA_OK
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = ws.data_ptr(), n
    torch.cuda.synchronize()
    assert capi.quant_fwd(p) == capi.FA_OK, capi.last_error()
    torch.cuda.synchronize()
    assert (out[total:] == 7).all() and (lse[4 * total:] == 7).all()
    lse = lse[:4 * total].view(4, total)
    at = 0
    for b, m in enumerate(left):
        if m:
            check_attend(out[at:at + m], lse[:, at:at + m], q[at:at + m], *c.rows(b), torch.bfloat16, causal=causal)
        at += m


@pytest.mark.parametrize("new", [[4, 1, 3], [40, 30, 20]])
def test_a_step_with_too_small_a_total_new(new):
    """update_page_table, append and attention with room for all but the last two tokens."""
    print(f"case small total_new {new}", flush=True)
    g = torch.Generator().manual_seed(62)
    total, B, P, Hk, D = sum(new) - 2, len(new), 16, 2, 64
    table, free = torch.full((B, 8), -1, **I32), torch.arange(30, **I32)
    zero, lens = torch.zeros(B, **I32), torch.tensor(new, **I32)
    slots, cu, _ = fa.update_page_table(table, zero, lens, free, torch.tensor([30], **I32), P, total)
    assert cu.tolist() == [0] + torch.tensor(new).cumsum(0).tolist() and slots.shape == (total,)
    k, v = (torch.randn(total, Hk, D, generator=g).to(torch.bfloat16) for _ in range(2))
    kc, vc = (torch.full((30, P, Hk, D), 0x7f, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((30, 1, Hk), float("nan"), device=DEV) for _ in range(2))
    fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), kc, vc, ks, vs, slots)
    q = torch.randn(total, 4, D, generator=g).to(torch.bfloat16)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), kc, vc, ks, vs, lens, page_table=table, cu_seqlens_q=cu,
                                                    max_seqlen_q=max(new), causal=True, return_softmax_lse=True)
    from oracle import fa_quant_oracle as qo
    at = 0
    for b, n in enumerate(new):
        m = min(n, total - at)
        kk, ok = qo.rows_of(kc.cpu(), ks.cpu(), table[b].tolist(), m)
        vv, _ = qo.rows_of(vc.cpu(), vs.cpu(), table[b].tolist(), m)
        check_attend(out[at:at + m], lse[:, at:at + m], q[at:at + m], kk, vv, ok, 448 * 2.0 ** -6, torch.bfloat16, causal=True)
        at += m
    assert at == total
