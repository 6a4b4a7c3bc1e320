"""Prompts and chunks over a 4-bit cache by either way: few rows go in blocks of 32 through the kernel for single tokens, more,
or rows that read many keys, through the one for prompts. A ragged call whose q goes on behind its last sequence is one of
more rows, so the same sequences take both."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from tests._fp4 import TYPES, Cache4, check_attend4

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
LONG = 16384  # rows times heads from which a call has more than 512 blocks


def attend(c, q, rows, dtype, behind=0, **how):
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **I32)
    tail = torch.full((behind, *q.shape[1:]), float("nan"), dtype=q.dtype)
    kw = {("window_size" if k == "window" else k): v for k, v in how.items()}
    return fa.flash_attn_with_quantized_kvcache(torch.cat([q, tail]).to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32), page_table=c.table.to(DEV),
                                                cu_seqlens_q=cu, max_seqlen_q=max(rows), return_softmax_lse=True, **kw)


def check(c, q, rows, dtype, out, lse, **how):
    at = 0
    for b, n in enumerate(rows):
        if n:
            s = slice(at, at + n)
            check_attend4(out[s], lse[:, s], q[s], *c.rows(b, dtype), dtype, **how)
        at += n


@pytest.mark.parametrize("how", [dict(causal=True), dict(), dict(window=(70, 0)), dict(window=(17, 30)), dict(window=(-1, -20)),
                                 dict(window=(0, 0)), dict(causal=True, softcap=20.0)], ids=str)
@pytest.mark.parametrize("long", [False, True], ids=["blocks", "prompts"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_masks(D, dt, long, how):
    """Blocks that end in the middle of a token's heads (3 of them), that see no key at the start or the end of a sequence,
    single tokens and nothing among them."""
    print(f"case fp4 blocks {D} {dt} {long} {how}", flush=True)
    g = torch.Generator().manual_seed(51)
    rows = [70, 1, 0, 33, 11, 128]
    c = Cache4(g, [40, 300, 20, 700, 0, 333], 2, D, 48)
    q = torch.randn(sum(rows), 6, D, generator=g).to(TYPES[dt])
    out, lse = attend(c, q, rows, TYPES[dt], LONG // 6 if long else 0, **how)
    check(c, q, rows, TYPES[dt], out, lse, **how)


@pytest.mark.parametrize("H,Hk", [(1, 1), (5, 1), (40, 1), (8, 8), (24, 3), (32, 8)])
@pytest.mark.parametrize("long", [False, True], ids=["blocks", "prompts"])
def test_heads(H, Hk, long):
    print(f"case fp4 block heads {H} {Hk} {long}", flush=True)
    g = torch.Generator().manual_seed(52)
    rows = [90, 2, 41]
    c = Cache4(g, [500, 130, 41], Hk, 128, 32)
    q = torch.randn(sum(rows), H, 128, generator=g).to(torch.bfloat16)
    out, lse = attend(c, q, rows, torch.bfloat16, LONG // H if long else 0, causal=True)
    check(c, q, rows, torch.bfloat16, out, lse, causal=True)


@pytest.mark.parametrize("rows", [[128], [64, 1, 64], [40, 40, 40, 1, 1]])
def test_graph_takes_either_way(rows):
    """A captured call replayed with lengths on both sides of what blocks take: 128 tokens of 8 heads onto 2 are 2 * 32 pairs of block and head, up
    to 256 tiles of 64 keys each."""
    print(f"case fp4 block graph {rows}", flush=True)
    g = torch.Generator().manual_seed(53)
    most = [n + 20000 for n in rows]
    c = Cache4(g, most, 2, 64, 256)
    q = torch.randn(sum(rows), 8, 64, generator=g).to(torch.bfloat16)
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **I32)
    st = [q.to(DEV), *c.args(DEV), torch.tensor(most, **I32)]
    table = c.table.to(DEV)

    def call():
        return fa.flash_attn_with_quantized_kvcache(*st, page_table=table, cu_seqlens_q=cu, max_seqlen_q=max(rows), causal=True, return_softmax_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = call()
    for keys in ([20000] * 5, [30] * 5, [16000, 0, 20000, 1, 7], [9, 19000, 0, 0, 0], [16256] * 5, [20000] * 5):
        c.lens = [n + k for n, k in zip(rows, keys)]
        st[5].copy_(torch.tensor(c.lens, **I32))
        want = call()
        for t in res:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
        if max(keys) < 20000 or len(rows) == 1:
            check(c, q, rows, torch.bfloat16, *res, causal=True)


@pytest.mark.parametrize("B,sq,H,Hk", [(1, 500, 32, 8), (1, 513, 32, 8), (64, 33, 4, 1), (16, 33, 32, 8), (512, 9, 4, 1), (513, 9, 4, 1)])
def test_the_number_of_blocks(B, sq, H, Hk):
    """Dense calls of 500 to 544 pairs of block and head, and of the most sequences with blocks."""
    print(f"case fp4 number of blocks {B} {sq} {H} {Hk}", flush=True)
    g = torch.Generator().manual_seed(54)
    c = Cache4(g, [(b * 37) % 90 + (sq if B < 4 else 0) for b in range(B)], Hk, 64, 16)
    q = torch.randn(B, sq, H, 64, generator=g).to(torch.float16)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32), page_table=c.table.to(DEV), causal=True,
                                                    return_softmax_lse=True)
    for b in list(range(min(B, 9))) + [B - 1]:
        check_attend4(out[b], lse[b], q[b], *c.rows(b, torch.float16), torch.float16, causal=True)


@pytest.mark.parametrize("rows,keys,behind", [([64, 1, 70, 3], [9000, 12000, 4000, 16000], 0), ([1], [30000], 40), ([3], [9], 40), ([40, 4], [20000, 20000], 0),
                                              ([5, 5, 0], [300, 40000, 7], 60)])
@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_beside_long_keys(D, rows, keys, behind):
    """Single tokens beside prompts whose keys are too many for blocks; padded calls of fewer rows than they are sized for."""
    print(f"case fp4 few rows beside long keys {D} {rows}", flush=True)
    g = torch.Generator().manual_seed(55)
    c = Cache4(g, keys, 2, D, 128)
    q = torch.randn(sum(rows), 8, D, generator=g).to(torch.bfloat16)
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **I32)
    tail = torch.full((behind, 8, D), float("nan"), dtype=q.dtype)
    out, lse = fa.flash_attn_with_quantized_kvcache(torch.cat([q, tail]).to(DEV), *c.args(DEV), torch.tensor(c.lens, **I32),
                                                    page_table=c.table.to(DEV), cu_seqlens_q=cu, max_seqlen_q=max(*rows, 16), causal=True,
                                                    return_softmax_lse=True)
    check(c, q, rows, torch.bfloat16, out, lse, causal=True)
