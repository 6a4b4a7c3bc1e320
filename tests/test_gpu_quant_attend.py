"""flash_attn_with_quantized_kvcache against its 64-bit definition. Every row,
scale and page id that a call may not use is NaN, the largest code or out of range."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._quant import TYPES, Cache, check_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def run(c, q, **kw):
    table = None if c.table is None else c.table.to(DEV)
    return fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32), page_table=table,
                                                return_softmax_lse=True, **kw)


def check(c, q, dtype, out, lse, **how):
    for b in range(len(c.lens)):
        check_attend(out[b], lse[b], q[b], *c.rows(b), dtype, **how)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (64, 64), (80, 80), (256, 64), (0, 128)])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_decode_lengths_and_pages(dt, cache, page, block):
    print(f"case decode {dt} {cache} {page}/{block}", flush=True)
    g = torch.Generator().manual_seed(1)
    c = Cache(g, [0, 1, 16, 63, 65, 777, 1300], 2, 128, cache, page, block, room=1408)
    q = torch.randn(7, 1, 8, 128, generator=g).to(TYPES[dt])
    out, lse = run(c, q, causal=True)
    check(c, q, TYPES[dt], out, lse, causal=True)


@pytest.mark.parametrize("D", [16, 48, 64, 80, 112, 128, 144, 192, 256])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("sq", [1, 3, 40])
def test_head_dims(D, cache, sq):
    print(f"case head dim {D} {cache} {sq}", flush=True)
    g = torch.Generator().manual_seed(2)
    c = Cache(g, [333, 40, 5], 2, D, cache, 32, 16)
    q = torch.randn(3, sq, 6, D, generator=g).to(torch.bfloat16)
    out, lse = run(c, q, causal=True)
    check(c, q, torch.bfloat16, out, lse, causal=True)


@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 4), (5, 5), (6, 2), (8, 1), (24, 3), (16, 1), (40, 1), (32, 8)])
@pytest.mark.parametrize("sq", [1, 2, 7])
def test_heads_and_rows(H, Hk, sq):
    """1 to 280 packed rows a key / value head."""
    print(f"case heads {H}/{Hk} rows {sq}", flush=True)
    g = torch.Generator().manual_seed(3)
    c = Cache(g, [300, 129], Hk, 64, "int8", 64, 32)
    q = torch.randn(2, sq, H, 64, generator=g).to(torch.float16)
    out, lse = run(c, q, causal=True)
    check(c, q, torch.float16, out, lse, causal=True)


@pytest.mark.parametrize("sq", [1, 5, 70])
@pytest.mark.parametrize("how", [dict(), dict(causal=True), dict(window=(100, 0)), dict(window=(17, 30)),
                                 dict(window=(-1, 3)), dict(window=(0, 0)), dict(causal=True, softcap=20.0),
                                 dict(window=(64, 0), softcap=5.0)], ids=str)
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_masks(cache, how, sq):
    """Lengths below the query rows too: rows that see no key."""
    print(f"case masks {cache} {how} {sq}", flush=True)
    g = torch.Generator().manual_seed(4)
    c = Cache(g, [0, 3, 64, 261, 600], 2, 128, cache, 64, 16)
    q = torch.randn(5, sq, 4, 128, generator=g).to(torch.bfloat16)
    kw = dict(how)
    out, lse = run(c, q, **{("window_size" if k == "window" else k): v for k, v in kw.items()})
    check(c, q, torch.bfloat16, out, lse, **how)


@pytest.mark.parametrize("lens", [[1, 1, 1], [1, 200, 0, 3, 1], [64, 1], [300, 300]])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_ragged_queries(cache, lens):
    """Decoding and prompt rows in one call; rows behind the last sequence stay as they are."""
    print(f"case ragged {cache} {lens}", flush=True)
    g = torch.Generator().manual_seed(5)
    c = Cache(g, [n + 37 * i for i, n in enumerate(lens)], 2, 128, cache, 128, 32)
    total = sum(lens)
    q = torch.randn(total + 3, 8, 128, generator=g).to(torch.bfloat16)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], **I32)
    out, lse = run(c, q, causal=True, cu_seqlens_q=cu, max_seqlen_q=max(lens))
    at = 0
    for b, n in enumerate(lens):
        check_attend(out[at:at + n], lse[:, at:at + n], q[at:at + n], *c.rows(b), torch.bfloat16, causal=True)
        at += n


def test_rows_behind_the_last_sequence_are_left():
    from fa_mi355x import capi
    print("case rows behind the last sequence", flush=True)
    g = torch.Generator().manual_seed(6)
    c = Cache(g, [50], 1, 64, "int8", 64, 64)
    q = torch.randn(40, 2, 64, generator=g).to(torch.float16).to(DEV)
    out = torch.full_like(q, 7.0)
    lse = torch.full((2, 40), 7.0, device=DEV)
    k, v, ks, vs = c.args(DEV)
    cu, lens, table = torch.tensor([0, 33], **I32), torch.tensor([50], **I32), c.table.to(DEV)
    p = capi.new_quant_fwd_params(
        dtype=capi.FA_DTYPE_FP16, cache_dtype=capi.FA_DTYPE_INT8, batch=1, seqlen_q=33, nheads=2, nheads_k=1, headdim=64,
        num_pages=k.shape[0], page_size=64, scale_block=64, q=q.data_ptr(), q_row_stride=128, q_head_stride=64,
        k=k.data_ptr(), k_page_stride=64 * 64, k_row_stride=64, k_head_stride=64,
        v=v.data_ptr(), v_page_stride=64 * 64, v_row_stride=64, v_head_stride=64,
        k_scale=ks.data_ptr(), k_scale_page_stride=1, k_scale_block_stride=1, k_scale_head_stride=1,
        v_scale=vs.data_ptr(), v_scale_page_stride=1, v_scale_block_stride=1, v_scale_head_stride=1,
        out=out.data_ptr(), out_row_stride=128, out_head_stride=64, softmax_lse=lse.data_ptr(),
        cache_seqlens=lens.data_ptr(), cu_seqlens_q=cu.data_ptr(), total_q=40, page_table=table.data_ptr(),
        page_table_row_stride=table.shape[1], table_rows=1, max_pages=table.shape[1], softmax_scale=0.125, is_causal=1)
    st, n = capi.quant_fwd_workspace_size(p)
    assert st == capi.FA_OK
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = ws.data_ptr(), n
    torch.cuda.synchronize()
    assert capi.quant_fwd(p) == capi.FA_OK, capi.last_error()
    torch.cuda.synchronize()
    check_attend(out[:33], lse[:, :33], q[:33].cpu(), *c.rows(0), torch.float16, causal=True)
    assert (out[33:] == 7).all() and (lse[:, 33:] == 7).all()


@pytest.mark.parametrize("sq", [1, 30])
def test_pages_outside_the_cache_are_not_visible(sq):
    print(f"case bad pages {sq}", flush=True)
    g = torch.Generator().manual_seed(7)
    c = Cache(g, [500, 130], 2, 128, "e4m3", 32, 32)
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
    print(f"case cache_batch_idx {page} {sq}", flush=True)
    g = torch.Generator().manual_seed(8)
    c = Cache(g, [256, 100, 199], 2, 64, "int8", page, 32, room=256)
    idx = [2, 0]
    q = torch.randn(2, sq, 8, 64, generator=g).to(torch.bfloat16)
    out, lse = fa.flash_attn_with_quantized_kvcache(
        q.to(DEV), *c.args(DEV), torch.tensor([c.lens[i] for i in idx], **I32), causal=True, return_softmax_lse=True,
        page_table=None if c.table is None else c.table.to(DEV), cache_batch_idx=torch.tensor(idx, **I32))
    for b, i in enumerate(idx):
        check_attend(out[b], lse[b], q[b], *c.rows(i), torch.bfloat16, causal=True)


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("sq", [1, 50])
def test_strides(cache, sq):
    """Queries out of a fused projection, caches that interleave K and V, heads outermost, transposed scales,
    a page table out of a wider one."""
    print(f"case strides {cache} {sq}", flush=True)
    g = torch.Generator().manual_seed(9)
    c = Cache(g, [270, 64], 2, 128, cache, 32, 16)
    qkv = torch.randn(2, sq, 12, 128, generator=g).to(torch.bfloat16).to(DEV)
    q = qkv[:, :, 2:10]
    k, v, ks, vs = c.args(DEV)
    n = k.shape[0]
    both = torch.empty(n, 2, 2, 32, 128, dtype=torch.uint8, device=DEV)  # page, k / v, head, row, dim
    both[:, 0] = k.view(torch.uint8).transpose(1, 2)
    both[:, 1] = v.view(torch.uint8).transpose(1, 2)
    kv = [both[:, i].transpose(1, 2).view(k.dtype) for i in (0, 1)]
    scales = [s.permute(2, 0, 1).contiguous().permute(1, 2, 0) for s in (ks, vs)]
    table = torch.nn.functional.pad(c.table, (0, 5)).to(DEV)[:, :c.table.shape[1]]
    out, lse = fa.flash_attn_with_quantized_kvcache(q, *kv, *scales, torch.tensor(c.lens, **I32), page_table=table,
                                                    causal=True, return_softmax_lse=True)
    for b in range(2):
        check_attend(out[b], lse[b], q[b].cpu(), *c.rows(b), torch.bfloat16, causal=True)


@pytest.mark.parametrize("sq", [1, 33])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_scales_and_queries_of_any_size(dt, cache, sq):
    """Scales over 2^-20 .. 2^6 side by side, query rows over 2^-12 .. 2^8."""
    print(f"case sizes {dt} {cache} {sq}", flush=True)
    g = torch.Generator().manual_seed(10)
    c = Cache(g, [400, 90], 2, 64, cache, 64, 16)
    for s in c.scales:
        s.mul_(2.0 ** torch.randint(-15, 8, s.shape, generator=g))
    c.scales[0].mul_(2.0 ** -6)
    q = torch.randn(2, sq, 4, 64, generator=g) * 2.0 ** torch.randint(-12, 9, (2, sq, 4, 1), generator=g)
    q = q.to(TYPES[dt])
    out, lse = run(c, q)
    check(c, q, TYPES[dt], out, lse)


def test_zero_scales_and_a_zero_softmax_scale():
    print("case zero scales", flush=True)
    g = torch.Generator().manual_seed(11)
    for sq in (1, 20):
        c = Cache(g, [200], 1, 64, "int8", 64, 16)
        c.scales[0][:, 1] = 0
        c.scales[1][:, 2:] = 0
        q = torch.randn(1, sq, 4, 64, generator=g).to(torch.float16)
        out, lse = run(c, q)
        check(c, q, torch.float16, out, lse)
        out, lse = run(c, q, softmax_scale=0.0)
        check(c, q, torch.float16, out, lse, scale=0.0)
        out, lse = run(c, q, softmax_scale=-0.3)
        check(c, q, torch.float16, out, lse, scale=-0.3)


def test_many_sequences():
    """More sequences than one launch lists."""
    print("case many sequences", flush=True)
    g = torch.Generator().manual_seed(12)
    B = 2100
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    c = Cache(g, lens, 1, 16, "int8", 16, 16)
    for sq in (1, 20):
        q = torch.randn(B, sq, 2, 16, generator=g).to(torch.float16)
        out, lse = run(c, q, causal=True)
        for b in list(range(0, B, 97)) + [2047, 2048, 2049, B - 1]:
            check_attend(out[b], lse[b], q[b], *c.rows(b), torch.float16, causal=True)
        cu = torch.arange(0, (B + 1) * sq, sq, **I32)
        out2, lse2 = run(c, q.view(B * sq, 2, 16), causal=True, cu_seqlens_q=cu, max_seqlen_q=sq)
        assert torch.equal(out2.view_as(out), out)


def test_empty_calls():
    print("case empty calls", flush=True)
    g = torch.Generator().manual_seed(13)
    c = Cache(g, [20], 1, 64, "int8", 64, 64)
    out, lse = run(c, torch.zeros(1, 0, 2, 64, dtype=torch.float16))
    assert out.shape == (1, 0, 2, 64) and lse.shape == (1, 2, 0)
    out, lse = run(c, torch.zeros(0, 2, 64, dtype=torch.float16), cu_seqlens_q=torch.zeros(2, **I32), max_seqlen_q=0)
    assert out.shape == (0, 2, 64)


@pytest.mark.parametrize("sq", [1, 20])
def test_offsets_past_32_bits(sq):
    """A pool of more than 4 GiB: the first and the last of its pages."""
    print(f"case offsets past 32 bits {sq}", flush=True)
    g = torch.Generator().manual_seed(14)
    n, P, Hk, D = 36000, 128, 8, 128
    k = torch.zeros(n, P, Hk, D, dtype=torch.int8, device=DEV)
    v = torch.zeros(n, P, Hk, D, dtype=torch.int8, device=DEV)
    ks = torch.full((n, 1, Hk), 0.02, device=DEV)
    vs = torch.full((n, 1, Hk), 0.03, device=DEV)
    c = Cache(g, [2 * P], Hk, D, "int8", P, P)
    pages = [0, n - 1]
    for at, page in zip(c.pages[0], pages):
        k[page], v[page], ks[page], vs[page] = (x[at].to(DEV) for x in (*c.codes, *c.scales))
    q = torch.randn(1, sq, 8, D, generator=g).to(torch.bfloat16)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), k, v, ks, vs, torch.tensor([2 * P], **I32),
                                                    page_table=torch.tensor([pages], **I32), return_softmax_lse=True)
    check_attend(out[0], lse[0], q[0], *c.rows(0), torch.bfloat16)


def test_long_contiguous_sequence_past_32_bits():
    """One sequence whose rows lie further apart than 2^31 bytes."""
    print("case long contiguous sequence", flush=True)
    g = torch.Generator().manual_seed(15)
    S, Hk, D = 24 << 20, 1, 128
    k = torch.zeros(1, S, Hk, D, dtype=torch.int8, device=DEV)
    v = torch.zeros(1, S, Hk, D, dtype=torch.int8, device=DEV)
    v[0, -1] = torch.randint(-127, 128, (Hk, D), generator=g).to(torch.int8)
    ks = torch.full((1, 1, Hk), 0.02, device=DEV)
    q = torch.randn(1, 1, 1, D, generator=g).to(torch.float16)
    # the window leaves the last 5 keys: zero scores, a fifth of the last value
    out = fa.flash_attn_with_quantized_kvcache(q.to(DEV), k, v, ks, ks, torch.tensor([S], **I32), causal=True,
                                               window_size=(4, 0))
    want = v[0, -1].double() * ks[0, 0, 0].double() / 5
    assert ((out[0, 0].double() - want).abs() <= 2.0 ** -10 * want.abs()).all()


@pytest.mark.parametrize("sq", [1, 24])
def test_graph_and_streams(sq):
    """Captured calls replayed with other lengths and codes, eager work between; two graphs at once; another stream."""
    print(f"case graphs {sq}", flush=True)
    g = torch.Generator().manual_seed(16)
    cs = [Cache(g, [300, 41], 2, 128, "e4m3", 64, 32) for _ in range(2)]
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
            check_attend(eager[0][b], eager[1][b], q[b], *c.rows(b), torch.bfloat16, causal=True)
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
    print(f"case repeated {sq}", flush=True)
    g = torch.Generator().manual_seed(17)
    c = Cache(g, [2000, 15, 900], 4, 128, "int8", 64, 64)
    q = torch.randn(3, sq, 16, 128, generator=g).to(torch.bfloat16)
    a = run(c, q, causal=True)
    for _ in range(3):
        b = run(c, q, causal=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
