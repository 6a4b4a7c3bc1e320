"""flash_attn_with_quantized_kvcache over a 4-bit cache against its 64-bit definition. Every row,
scale and page id that a call may not use is NaN or out of range."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import capi
from oracle import fa_fp4_oracle as fo
from tests._fp4 import TYPES, Cache4, check_attend4

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def run(c, q, **kw):
    table = None if c.table is None else c.table.to(DEV)
    return fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32), page_table=table,
                                                return_softmax_lse=True, **kw)


def check(c, q, dtype, out, lse, **how):
    for b in range(len(c.lens)):
        check_attend4(out[b], lse[b], q[b], *c.rows(b, dtype), dtype, **how)


@pytest.mark.parametrize("page", [16, 48, 64, 80, 256, 0])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_lengths_and_pages(dt, page, D):
    print(f"case fp4 decode {dt} {page} {D}", flush=True)
    g = torch.Generator().manual_seed(1)
    c = Cache4(g, [0, 1, 16, 63, 65, 777, 1300], 2, D, page, room=1312)
    q = torch.randn(7, 1, 8, D, generator=g).to(TYPES[dt])
    out, lse = run(c, q, causal=True)
    check(c, q, TYPES[dt], out, lse, causal=True)


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("sq", [1, 3, 40, 150])
def test_head_dims(D, dt, sq):
    print(f"case fp4 head dim {D} {dt} {sq}", flush=True)
    g = torch.Generator().manual_seed(2)
    c = Cache4(g, [333, 40, 5], 2, D, 32)
    q = torch.randn(3, sq, 6, D, generator=g).to(TYPES[dt])
    out, lse = run(c, q, causal=True)
    check(c, q, TYPES[dt], out, lse, causal=True)


@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 4), (5, 5), (6, 2), (8, 1), (24, 3), (16, 1), (40, 1), (32, 8)])
@pytest.mark.parametrize("sq", [1, 2, 7])
def test_heads_and_rows(H, Hk, sq):
    """1 to 280 packed rows a key / value head."""
    print(f"case fp4 heads {H}/{Hk} rows {sq}", flush=True)
    g = torch.Generator().manual_seed(3)
    c = Cache4(g, [300, 129], Hk, 64, 64)
    q = torch.randn(2, sq, H, 64, generator=g).to(torch.float16)
    out, lse = run(c, q, causal=True)
    check(c, q, torch.float16, out, lse, causal=True)


@pytest.mark.parametrize("sq", [1, 5, 70])
@pytest.mark.parametrize("how", [dict(), dict(causal=True), dict(window=(100, 0)), dict(window=(17, 30)),
                                 dict(window=(-1, 3)), dict(window=(0, 0)), dict(causal=True, softcap=20.0),
                                 dict(window=(64, 0), softcap=5.0)], ids=str)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_masks(dt, how, sq):
    """Lengths below the query rows too: rows that see no key."""
    print(f"case fp4 masks {dt} {how} {sq}", flush=True)
    g = torch.Generator().manual_seed(4)
    c = Cache4(g, [0, 3, 64, 261, 600], 2, 128, 64)
    q = torch.randn(5, sq, 4, 128, generator=g).to(TYPES[dt])
    out, lse = run(c, q, **{("window_size" if k == "window" else k): v for k, v in how.items()})
    check(c, q, TYPES[dt], out, lse, **how)


@pytest.mark.parametrize("lens", [[1, 1, 1], [1, 200, 0, 3, 1], [64, 1], [300, 300]])
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_queries(D, lens):
    """Decoding and prompt rows in one call."""
    print(f"case fp4 ragged {D} {lens}", flush=True)
    g = torch.Generator().manual_seed(5)
    c = Cache4(g, [n + 37 * i for i, n in enumerate(lens)], 2, D, 128)
    total = sum(lens)
    q = torch.randn(total + 3, 8, D, generator=g).to(torch.bfloat16)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], **I32)
    out, lse = run(c, q, causal=True, cu_seqlens_q=cu, max_seqlen_q=max(lens))
    at = 0
    for b, n in enumerate(lens):
        check_attend4(out[at:at + n], lse[:, at:at + n], q[at:at + n], *c.rows(b, torch.bfloat16), torch.bfloat16, causal=True)
        at += n


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("Hk,lens", [(2, [700, 3, 40, 0, 129, 1, 260]), (8, [300, 300, 300]), (1, [1100])])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cut_items(D, Hk, lens, dt):
    """Ragged batches whose items the workgroups share, over several groups of 1024 keys."""
    print(f"case fp4 cut {D} {Hk} {lens} {dt}", flush=True)
    g = torch.Generator().manual_seed(22)
    keys = [n + (1900 if i % 3 == 0 else 5) for i, n in enumerate(lens)]
    c = Cache4(g, keys, Hk, D, 32)
    q = torch.randn(sum(lens), 2 * Hk, D, generator=g).to(TYPES[dt])
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    out, lse = run(c, q, cu_seqlens_q=cu.to(DEV), max_seqlen_q=max(lens), causal=True)
    for b, n in enumerate(lens):
        if n:
            r = slice(int(cu[b]), int(cu[b + 1]))
            check_attend4(out[r], lse[:, r], q[r], *c.rows(b, TYPES[dt]), TYPES[dt], causal=True)


def c_call(c, q, lens, rows, total, dtype, causal=True, **more):
    """The C entry on buffers that go on behind total_q; (out, lse) as they are after it, filled with 7 before."""
    D, Hk = q.shape[2], c.codes[0].shape[2]
    qd = q.to(DEV)
    out, lse = torch.full_like(qd, 7.0), torch.full((q.shape[1] * total + q.shape[0],), 7.0, device=DEV)
    dev = c.args(DEV)
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **I32)
    table = torch.nn.functional.pad(c.table, (0, 6), value=0x7fffffff).to(DEV)
    lens = torch.tensor(lens, **I32)
    f = {}
    for name, t in zip(("k", "v", "k_scale", "v_scale"), dev):
        row = "block" if "scale" in name else "row"
        f.update({name: t.data_ptr(), name + "_page_stride": t.stride(0), f"{name}_{row}_stride": t.stride(1), name + "_head_stride": t.stride(2)})
    p = capi.new_quant_fwd_params(
        dtype=capi.FA_DTYPE_BF16 if dtype == torch.bfloat16 else capi.FA_DTYPE_FP16, cache_dtype=capi.FA_DTYPE_FP4_E2M1, batch=len(rows),
        seqlen_q=max(rows), nheads=q.shape[1], nheads_k=Hk, headdim=D, num_pages=dev[0].shape[0], page_size=c.page, scale_block=1,
        q=qd.data_ptr(), q_row_stride=qd.stride(0), q_head_stride=D, **f, out=out.data_ptr(), out_row_stride=out.stride(0), out_head_stride=D,
        softmax_lse=lse.data_ptr(), cache_seqlens=lens.data_ptr(), cu_seqlens_q=cu.data_ptr(), total_q=total, page_table=table.data_ptr(),
        page_table_row_stride=table.shape[1], table_rows=len(rows), max_pages=table.shape[1], softmax_scale=D ** -0.5, is_causal=int(causal), **more)
    st, n = capi.fp4_fwd_workspace_size(p)
    assert st == capi.FA_OK
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = ws.data_ptr(), n
    torch.cuda.synchronize()
    assert capi.fp4_fwd(p) == capi.FA_OK, capi.last_error()
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,total", [([3, 5, 2], 10), ([33], 33), ([3, 5, 2], 6), ([2, 2, 2], 2), ([40, 60, 3], 77), ([1, 90, 0, 1], 91), ([300, 20], 299)])
def test_rows_past_the_end(rows, total, causal):
    """Rows behind the last sequence and behind total_q are neither read nor written; the others keep their positions."""
    print(f"case fp4 rows past the end {rows} {total} {causal}", flush=True)
    g = torch.Generator().manual_seed(61)
    have = [700, 20, 31, 5][:len(rows)]
    left = [max(0, min(sum(rows[:i + 1]), total) - min(sum(rows[:i]), total)) for i in range(len(rows))]
    c = Cache4(g, [h + n for h, n in zip(have, left)], 2, 64, 16)  # keys of dropped tokens: poisoned or no page
    q = torch.full((sum(rows) + 5, 4, 64), float("nan"), dtype=torch.bfloat16)
    q[:total] = torch.randn(total, 4, 64, generator=g).to(torch.bfloat16)
    out, lse = c_call(c, q, [h + n for h, n in zip(have, rows)], rows, total, torch.bfloat16, causal)
    assert (out[total:] == 7).all() and (lse[4 * total:] == 7).all()
    lse = lse[:4 * total].view(4, total)
    at = 0
    for b, m in enumerate(left):
        if m:
            check_attend4(out[at:at + m], lse[:, at:at + m], q[at:at + m], *c.rows(b, torch.bfloat16), torch.bfloat16, causal=causal)
        at += m


@pytest.mark.parametrize("sq", [1, 30])
def test_pages_outside_the_cache_are_not_visible(sq):
    print(f"case fp4 bad pages {sq}", flush=True)
    g = torch.Generator().manual_seed(7)
    c = Cache4(g, [500, 130], 2, 128, 32)
    c.table[0, 2] = -1
    c.table[0, 7] = c.codes[0].shape[0]
    c.table[0, 15] = 1 << 30  # holds the last keys
    c.table[1, :] = -5        # a sequence without any page
    q = torch.randn(2, sq, 4, 128, generator=g).to(torch.bfloat16)
    out, lse = run(c, q, causal=True)
    check(c, q, torch.bfloat16, out, lse, causal=True)


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("sq", [1, 24])
def test_cache_batch_idx(page, sq):
    """Rows of other requests, rows that are not there, and the same row twice."""
    print(f"case fp4 cache_batch_idx {page} {sq}", flush=True)
    g = torch.Generator().manual_seed(8)
    c = Cache4(g, [256, 100, 199], 2, 64, page, room=256)
    idx = [2, 0, 7, 2, -1]
    q = torch.randn(5, sq, 8, 64, generator=g).to(torch.bfloat16)
    lens = [c.lens[i] if 0 <= i < 3 else 50 for i in idx]
    out, lse = fa.flash_attn_with_quantized_kvcache(
        q.to(DEV), *c.args(DEV), torch.tensor(lens, **I32), causal=True, return_softmax_lse=True,
        page_table=None if c.table is None else c.table.to(DEV), cache_batch_idx=torch.tensor(idx, **I32))
    for b, i in enumerate(idx):
        if 0 <= i < 3:
            check_attend4(out[b], lse[b], q[b], *c.rows(i, torch.bfloat16), torch.bfloat16, causal=True)
        else:
            assert not out[b].any() and (lse[b] == float("inf")).all()


@pytest.mark.parametrize("sq", [1, 50])
def test_strides(sq):
    """Queries out of a fused projection, caches that interleave K and V, heads outermost, scales beside each other, a page table
    out of a wider one."""
    print(f"case fp4 strides {sq}", flush=True)
    g = torch.Generator().manual_seed(9)
    c = Cache4(g, [270, 64], 2, 128, 32)
    q = torch.randn(2, sq, 12, 128, generator=g).to(torch.bfloat16).to(DEV)[:, :, 2:10]
    k, v, ks, vs = c.args(DEV)
    n = k.shape[0]
    both = torch.empty(n, 2, 2, 32, 64, dtype=torch.uint8, device=DEV)  # page, k / v, head, row, byte
    both[:, 0], both[:, 1] = k.transpose(1, 2), v.transpose(1, 2)
    scales = torch.empty(2, n, 32, 9, dtype=torch.uint8, device=DEV)  # head, page, row, odd number of bytes
    kv = [both[:, i].transpose(1, 2) for i in (0, 1)]
    sc = [scales[..., 1 + 4 * i:5 + 4 * i].permute(1, 2, 0, 3) for i in (0, 1)]
    sc[0].copy_(ks)
    sc[1].copy_(vs)
    table = torch.nn.functional.pad(c.table, (0, 5)).to(DEV)[:, :c.table.shape[1]]
    out, lse = fa.flash_attn_with_quantized_kvcache(q, *kv, *sc, torch.tensor(c.lens, **I32), page_table=table,
                                                    causal=True, return_softmax_lse=True)
    for b in range(2):
        check_attend4(out[b], lse[b], q[b].cpu(), *c.rows(b, torch.bfloat16), torch.bfloat16, causal=True)


@pytest.mark.parametrize("sq", [1, 33])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_scales_and_queries_of_any_size(dt, D, sq):
    """Scales over the range of the type side by side, V's above all; query rows over 2^-12 .. 2^8."""
    print(f"case fp4 sizes {dt} {D} {sq}", flush=True)
    g = torch.Generator().manual_seed(10)
    c = Cache4(g, [400, 90], 2, D, 64)
    lo, hi = (100, 141) if dt == "fp16" else (20, 240)
    for i, s in enumerate(c.scales):
        some = torch.randint(lo, hi, s.shape, generator=g, dtype=torch.uint8) if i else torch.randint(105, 128, s.shape, generator=g, dtype=torch.uint8)
        s.copy_(torch.where(s == 255, s, some))
    q = torch.randn(2, sq, 4, D, generator=g) * 2.0 ** torch.randint(-12, 9, (2, sq, 4, 1), generator=g)
    q = q.to(TYPES[dt])
    out, lse = run(c, q)
    check(c, q, TYPES[dt], out, lse)
    out, lse = run(c, q, softmax_scale=0.0)
    check(c, q, TYPES[dt], out, lse, scale=0.0)
    out, lse = run(c, q, softmax_scale=-0.003)
    check(c, q, TYPES[dt], out, lse, scale=-0.003)


@pytest.mark.parametrize("sq,seen", [(4, 62), (40, 300), (200, 333)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_that_are_no_numbers(sq, seen, which):
    """A NaN scale of a key reaches every row that sees it; of k (and of v where none of the call's rows sees it) no other."""
    print(f"case fp4 nan {sq} {seen} {which}", flush=True)
    g = torch.Generator().manual_seed(21)
    sk = seen + 2 if which == "k" else seen
    c = Cache4(g, [sk], 2, 64, 16)
    kk, vv, ok = c.rows(0, torch.bfloat16)
    at = c.pages[0][(sk - 1) // 16], (sk - 1) % 16
    (c.scales[0] if which == "k" else c.scales[1])[at] = 255
    q = torch.randn(1, sq, 4, 64, generator=g).to(torch.bfloat16)
    if which == "k":
        out, lse = run(c, q, causal=True)
        n = sq - 1  # only the last query sees the last key
        check_attend4(out[0, :n], lse[0, :, :n], q[0, :n], kk[:-1], vv[:-1], ok[:-1], torch.bfloat16, causal=True)
        assert torch.isnan(out[0, n:]).all() and torch.isnan(lse[0, :, n:]).all()
    else:
        out, lse = run(c, q)  # every row sees it
        assert torch.isnan(out).all()
        lens = torch.tensor([sk - 1], **I32)  # none does
        out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), lens, page_table=c.table.to(DEV), causal=True,
                                                        return_softmax_lse=True)
        check_attend4(out[0], lse[0], q[0], kk[:-1], vv[:-1], ok[:-1], torch.bfloat16, causal=True)


def test_many_sequences():
    """More sequences than one launch lists."""
    print("case fp4 many sequences", flush=True)
    g = torch.Generator().manual_seed(12)
    B = 2100
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    c = Cache4(g, lens, 1, 32, 16)
    for sq in (1, 20):
        q = torch.randn(B, sq, 2, 32, generator=g).to(torch.float16)
        out, lse = run(c, q, causal=True)
        for b in list(range(0, B, 97)) + [2047, 2048, 2049, B - 1]:
            check_attend4(out[b], lse[b], q[b], *c.rows(b, torch.float16), torch.float16, causal=True)
        cu = torch.arange(0, (B + 1) * sq, sq, **I32)
        out2, _ = run(c, q.view(B * sq, 2, 32), causal=True, cu_seqlens_q=cu, max_seqlen_q=sq)
        assert torch.equal(out2.view_as(out), out)


def test_empty_calls():
    print("case fp4 empty calls", flush=True)
    g = torch.Generator().manual_seed(13)
    c = Cache4(g, [20], 1, 64, 16)
    out, lse = run(c, torch.zeros(1, 0, 2, 64, dtype=torch.float16))
    assert out.shape == (1, 0, 2, 64) and lse.shape == (1, 2, 0)
    out, lse = run(c, torch.zeros(0, 2, 64, dtype=torch.float16), cu_seqlens_q=torch.zeros(2, **I32), max_seqlen_q=0)
    assert out.shape == (0, 2, 64)
    k, v = fa.read_quantized_kvcache(*c.args(DEV), slot_mapping=torch.zeros(0, dtype=torch.int64, device=DEV))
    assert k.shape == v.shape == (0, 1, 64)
    fa.append_quantized_kvcache(k, v, *c.args(DEV), torch.zeros(0, dtype=torch.int64, device=DEV))


@pytest.mark.parametrize("sq", [1, 20])
def test_offsets_past_32_bits(sq):
    """A pool of more than 4 GiB: the first and the last of its pages, attended to, appended to and read."""
    print(f"case fp4 offsets past 32 bits {sq}", flush=True)
    g = torch.Generator().manual_seed(14)
    n, P, Hk, D = 72000, 128, 8, 128
    k, v = (torch.zeros(n, P, Hk, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((n, P, Hk, D // 32), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    c = Cache4(g, [2 * P], Hk, D, P)
    pages = [0, n - 1]
    for at, page in zip(c.pages[0], pages):
        k[page], v[page], ks[page], vs[page] = (x[at].to(DEV) for x in (*c.codes, *c.scales))
    q = torch.randn(1, sq, 8, D, generator=g).to(torch.bfloat16)
    table = torch.tensor([pages], **I32)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), k, v, ks, vs, torch.tensor([2 * P], **I32), page_table=table,
                                                    return_softmax_lse=True)
    check_attend4(out[0], lse[0], q[0], *c.rows(0, torch.bfloat16), torch.bfloat16)
    kk, vv, _ = c.rows(0, torch.bfloat16)
    got = fa.read_quantized_kvcache(k, v, ks, vs, cu_seqlens_k=torch.tensor([0, 2 * P], **I32), total_k=2 * P, page_table=table)
    assert torch.equal(got[0].cpu().double(), kk) and torch.equal(got[1].cpu().double(), vv)
    new = torch.randn(2, Hk, D, generator=g).to(torch.bfloat16)
    slots = torch.tensor([n * P - 1, 5], device=DEV)
    fa.append_quantized_kvcache(new.to(DEV), new.to(DEV), k, v, ks, vs, slots)
    want = [torch.zeros(1, 16, Hk, D // 2, dtype=torch.uint8), torch.zeros(1, 16, Hk, D // 32, dtype=torch.uint8)]
    fo.append(new, *want, [0, 1])
    for codes, sc in ((k, ks), (v, vs)):
        assert torch.equal(torch.stack((codes[-1, -1], codes[0, 5])).cpu(), want[0][0, :2])
        assert torch.equal(torch.stack((sc[-1, -1], sc[0, 5])).cpu(), want[1][0, :2])


def test_long_contiguous_sequence_past_32_bits():
    """One sequence whose rows lie further apart than 2^31 bytes."""
    print("case fp4 long contiguous sequence", flush=True)
    g = torch.Generator().manual_seed(15)
    S, Hk, D = 48 << 20, 1, 128
    k, v = (torch.zeros(1, S, Hk, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    s = torch.full((1, S, Hk, D // 32), 127, dtype=torch.uint8, device=DEV)
    v[0, -1] = torch.randint(0, 256, (Hk, D // 2), generator=g, dtype=torch.uint8)
    q = torch.randn(1, 1, 1, D, generator=g).to(torch.float16)
    # the window leaves the last 5 keys: zero scores, a fifth of the last value
    out = fa.flash_attn_with_quantized_kvcache(q.to(DEV), k, v, s, s, torch.tensor([S], **I32), causal=True, window_size=(4, 0))
    want = fo.values(v[0, -1].cpu(), s[0, -1].cpu()) / 5
    assert ((out[0, 0].cpu().double() - want).abs() <= 2.0 ** -10 * want.abs()).all()


@pytest.mark.parametrize("sq", [1, 24])
def test_graph_and_streams(sq):
    """Captured calls replayed with other lengths, eager work between; two graphs at once; another stream."""
    print(f"case fp4 graphs {sq}", flush=True)
    g = torch.Generator().manual_seed(16)
    cs = [Cache4(g, [300, 41], 2, 128, 64) for _ in range(2)]
    qs = [torch.randn(2, sq, 8, 128, generator=g).to(torch.bfloat16) for _ in range(2)]
    calls = []
    for c, q in zip(cs, qs):
        st = [*c.args(DEV), torch.tensor(c.lens, **I32)]
        qd, table = q.to(DEV), c.table.to(DEV)
        call = lambda st=st, qd=qd, table=table: fa.flash_attn_with_quantized_kvcache(  # noqa: E731
            qd, *st, page_table=table, causal=True, return_softmax_lse=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = call()
        torch.cuda.current_stream().wait_stream(side)
        for b in range(2):
            check_attend4(eager[0][b], eager[1][b], q[b], *c.rows(b, torch.bfloat16), torch.bfloat16, causal=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = call()
        calls.append((graph, res, st, call))
    for lens in ([300, 41], [17, 41], [300, 0], [250, 33]):
        for _, _, st, _ in calls:
            st[4].copy_(torch.tensor(lens, **I32))
        want = [[t.clone() for t in call()] for _, _, _, call in calls]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, res, _, _), s in zip(calls, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, res, _, _), w in zip(calls, want):
            assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])


@pytest.mark.parametrize("sq", [1, 3, 40])
def test_repeated_calls_agree_bit_for_bit(sq):
    print(f"case fp4 repeated {sq}", flush=True)
    g = torch.Generator().manual_seed(17)
    c = Cache4(g, [2000, 15, 900], 4, 128, 64)
    q = torch.randn(3, sq, 16, 128, generator=g).to(torch.bfloat16)
    a = run(c, q, causal=True)
    for _ in range(3):
        b = run(c, q, causal=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("sq", [1, 64])
def test_same_as_the_rows_read_back(sq):
    """Attention of the 16-bit kernels over read_quantized_kvcache's rows: two roundings of the weights apart."""
    print(f"case fp4 read and attend {sq}", flush=True)
    g = torch.Generator().manual_seed(18)
    c = Cache4(g, [500, 77], 2, 128, 32)
    q = torch.randn(2 * sq, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    cu_q = torch.tensor([0, sq, 2 * sq], **I32)
    cu_k = torch.tensor([0, 500, 577], **I32)
    out, lse = run(c, q, cu_seqlens_q=cu_q, max_seqlen_q=sq, causal=True)
    k, v = fa.read_quantized_kvcache(*c.args(DEV), cu_seqlens_k=cu_k, total_k=577, page_table=c.table.to(DEV))
    ref = fa.flash_attn_varlen_func(q, k, v, cu_q, cu_k, sq, 500, causal=True)
    size = fa.flash_attn_varlen_func(q, k, v.abs(), cu_q, cu_k, sq, 500, causal=True)
    # sum of p |v| times half a step for the weights of each, and half a step of each result
    assert ((out.float() - ref.float()).abs() <= size.float() * 2.0 ** -7 + ref.float().abs() * 2.0 ** -7 + 2.0 ** -12).all()
