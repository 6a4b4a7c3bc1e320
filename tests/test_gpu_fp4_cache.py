"""The 4-bit cache written and read back (append_quantized_kvcache, read_quantized_kvcache) against
oracle/fa_fp4_oracle.py: codes and scales byte for byte."""
import math
import random

import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_fp4_oracle as fo
from oracle import fa_quant_oracle as qo
from tests._fp4 import TYPES, Cache4, check_attend4
from tests._quant import Cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def empty_cache(g, pages, page, Hk, D):
    return [torch.randint(0, 256, (pages, page, Hk, w), generator=g, dtype=torch.uint8) for w in (D // 2, D // 2, D // 32, D // 32)]


def same_cache(dev, want):
    for d, w in zip(dev, want):
        assert torch.equal(d.cpu().view(torch.uint8), w)


def fill(x, kind, g):
    """Rows of a kind: plain ones, ones on the borders between two codes, extremes."""
    if kind == "ties":
        at = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 4.0, 7.0])
        y = at[torch.randint(0, len(at), x.shape, generator=g)] * torch.where(torch.rand(x.shape, generator=g) < 0.5, -1.0, 1.0)
        return y * 2.0 ** torch.randint(-9, 9, (*x.shape[:2], 1), generator=g)
    if kind == "extremes":
        e = torch.randint(-30, 17, x.shape, generator=g).double() if x.dtype == torch.float16 else \
            torch.randint(-133, 128, x.shape, generator=g).double()
        y = (x.double() * 2.0 ** e).clamp(-torch.finfo(x.dtype).max, torch.finfo(x.dtype).max)
        # whole groups of one size too, so that the largest scales and subnormal rows come up
        y[1::3] = x[1::3].double() * (2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -130)
        y[2::5] = torch.finfo(x.dtype).max
        y[4::7] = 0.0
        return y
    return x


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["plain", "ties", "extremes"])
@pytest.mark.parametrize("n,Hk,D,page", [(1, 1, 32, 16), (7, 2, 64, 16), (19, 3, 96, 48), (33, 1, 256, 32)])
def test_append(dtype, kind, n, Hk, D, page):
    print(f"case fp4 append {dtype} {kind} {n} {Hk} {D} {page}", flush=True)
    g = torch.Generator().manual_seed(n + D)
    dt, pages = TYPES[dtype], 6
    want = empty_cache(g, pages, page, Hk, D)
    dev = [t.to(DEV) for t in want]
    k, v = (fill(torch.randn(n, Hk, D, generator=g).to(dt), kind, g).to(dt) for _ in range(2))
    # slots in any order; some outside the cache
    at = torch.randperm(pages * page, generator=g)[:n]
    at[::5] = torch.tensor([-1, pages * page, 2 ** 40, -2 ** 62])[torch.arange(len(at[::5])) % 4]
    at[0] = at[0] if n > 1 else 3  # rows outside the cache alone write nothing
    fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), *dev, at.to(DEV))
    fo.append(k, want[0], want[2], at.tolist())
    fo.append(v, want[1], want[3], at.tolist())
    same_cache(dev, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_no_numbers(dtype):
    """+-inf count as the largest value, a NaN makes its group NaN and no other."""
    print(f"case fp4 append no numbers {dtype}", flush=True)
    g = torch.Generator().manual_seed(3)
    dt = TYPES[dtype]
    cache = [t.to(DEV) for t in empty_cache(g, 2, 16, 2, 64)]
    k = torch.randn(4, 2, 64, generator=g).to(dt)
    k[0, 0, 3], k[1, 1, 40], k[2, 0, 0], k[2, 0, 33] = math.inf, -math.inf, math.nan, math.inf
    fa.append_quantized_kvcache(k.to(DEV), k.to(DEV), *cache, torch.arange(4, device=DEV))
    got, _ = fa.read_quantized_kvcache(*cache, slot_mapping=torch.arange(4, device=DEV), dtype=torch.float32)
    got = got.cpu()
    nan = torch.zeros(4, 2, 64, dtype=torch.bool)
    nan[2, 0, :32] = True
    assert torch.equal(torch.isnan(got), nan)
    assert torch.isfinite(got[~nan]).all() and torch.isfinite(got[~nan].to(dt)).all()
    want = [torch.zeros(2, 16, 2, 32, dtype=torch.uint8), torch.zeros(2, 16, 2, 2, dtype=torch.uint8)]
    fo.append(k, *want, range(4))
    ref = fo.values(want[0][0, :4], want[1][0, :4])
    assert torch.equal(got[~nan].double(), ref[~nan])


def test_append_layouts():
    """Heads first, k and v of one tensor, caches that are parts of larger ones: strides of every kind; nothing else
    is written."""
    print("case fp4 append layouts", flush=True)
    g = torch.Generator().manual_seed(4)
    n, Hk, D, page = 9, 3, 64, 16
    both = torch.randn(Hk, n, 2, D, generator=g).to(torch.bfloat16)
    k, v = both[:, :, 0].transpose(0, 1), both[:, :, 1].transpose(0, 1)
    whole = torch.randint(0, 256, (5, 2, Hk + 1, page, D // 2), generator=g, dtype=torch.uint8)
    sc = torch.randint(0, 256, (5, page, 2, Hk, D // 32 + 3), generator=g, dtype=torch.uint8)
    view = lambda w, s: [w[:, 0, 1:].transpose(1, 2), w[:, 1, 1:].transpose(1, 2), s[:, :, 0, :, 1:3], s[:, :, 1, :, 1:3]]  # noqa: E731
    dev = [whole.to(DEV), sc.to(DEV)]
    at = torch.randperm(5 * page, generator=g)[:n]
    fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), *view(*dev), at.to(DEV))
    parts = view(whole, sc)
    fo.append(k, parts[0], parts[2], at.tolist())
    fo.append(v, parts[1], parts[3], at.tolist())
    assert torch.equal(dev[0].cpu(), whole) and torch.equal(dev[1].cpu(), sc)
    # rows of 16-bit values that a 16-byte load cannot take
    odd = torch.randn(n, Hk, D + 1, generator=g).to(torch.bfloat16)[:, :, 1:]
    fa.append_quantized_kvcache(odd.to(DEV), odd.to(DEV), *view(*dev), at.to(DEV))
    fo.append(odd, parts[0], parts[2], at.tolist())
    fo.append(odd, parts[1], parts[3], at.tolist())
    assert torch.equal(dev[0].cpu(), whole) and torch.equal(dev[1].cpu(), sc)


@pytest.mark.parametrize("n", [2047, 2049, 5000, 70000])
def test_append_many(n):
    """Counts of rows around those at which a workgroup takes more of them; values read back equal those of a plain
    quantisation by comparisons."""
    print(f"case fp4 append many {n}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(n)
    Hk, D, page = 2, 64, 16
    pages = -(-n // page)
    cache = [torch.zeros(pages, page, Hk, w, dtype=torch.uint8, device=DEV) for w in (D // 2, D // 2, D // 32, D // 32)]
    k, v = (torch.randn(n, Hk, D, generator=g, device=DEV).to(torch.float16) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n]
    fa.append_quantized_kvcache(k, v, *cache, slots)
    for got, x in zip(fa.read_quantized_kvcache(*cache, slot_mapping=slots, dtype=torch.float32), (k, v)):
        y = x.float().unflatten(-1, (-1, 32))
        m, e = torch.frexp(y.abs().amax(-1, keepdim=True))
        s = torch.exp2((e - 3 + (m > 0.75).int()).clamp(min=-100).float())
        a = y.abs() / s
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        r = torch.round(a / step) * step  # to even: of halves and of whole numbers that is the even code as well
        assert torch.equal(got, (torch.sign(y) * r.clamp(max=6) * s).flatten(-2))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
def test_read_every_value(out):
    """Every code under every scale, as the type holds it: nearest, ties to even, inf past the largest."""
    print(f"case fp4 read every value {out}", flush=True)
    codes = torch.arange(256, dtype=torch.uint8).view(16, 1, 1, 16).repeat(1, 256, 1, 1)
    scale = torch.arange(256, dtype=torch.uint8).view(1, 256, 1, 1).repeat(16, 1, 1, 1)
    dev = [t.to(DEV) for t in (codes, codes.flip(0), scale, scale)]
    slots = torch.arange(16 * 256, device=DEV)
    k, v = fa.read_quantized_kvcache(*dev, slot_mapping=slots, dtype=out)
    for got, c in ((k, codes), (v, codes.flip(0))):
        ref = fo.values(c, scale).flatten(0, 1).to(out)
        nan = torch.isnan(ref)
        got = got.cpu()
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], ref[~nan])


@pytest.mark.parametrize("cache,block", [("fp4", 1), ("int8", 16), ("e4m3", 48), ("e4m3", 16)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page,D,Hk", [(48, 96, 3), (0, 64, 1), (144, 256, 2)])
def test_read_sequences(cache, block, out, page, D, Hk):
    """Keys of sequences one behind the other, by slots too; rows behind the last one, missing pages and rows are 0."""
    print(f"case read {cache} {block} {out} {page} {D}", flush=True)
    g = torch.Generator().manual_seed(D)
    lens = [5, 0, 97, 1, 144]
    if cache == "fp4":
        c = Cache4(g, lens, Hk, D, page, room=144)
        one = lambda i, b: fo.rows_of(c.codes[i], c.scales[i], [b] if c.table is None else c.table[b].tolist(), lens[b])  # noqa: E731
    else:
        c = Cache(g, lens, Hk, D, cache, page, block, room=144)
        one = lambda i, b: qo.rows_of(c.codes[i], c.scales[i], [b] if c.table is None else c.table[b].tolist(), lens[b])  # noqa: E731
    if page:
        c.table[2, 1 if page < 97 else 0] = -1  # a missing page
    order = [2, 0, 4, 1, 3]
    n = [lens[b] for b in order]
    cu = [sum(n[:i]) for i in range(len(n) + 1)]
    more = dict(page_table=c.table.to(DEV)) if page else {}
    got = fa.read_quantized_kvcache(*c.args(DEV), cu_seqlens_k=i32(cu), total_k=cu[-1] + 3, cache_batch_idx=i32(order), dtype=out, **more)
    slots = []
    for b in order:
        for j in range(lens[b]):
            p = b if not page else c.table[b, j // page].item()
            slots.append(p * (page or 144) + j % (page or 144) if p >= 0 else -1)
    by_slot = fa.read_quantized_kvcache(*c.args(DEV), slot_mapping=torch.tensor(slots, device=DEV), dtype=out)
    for i in range(2):
        rows = []
        for b in order:
            x, ok = one(i, b)
            rows.append(torch.where(ok[:, None, None], x, 0.0))
        ref = torch.cat(rows).float().to(out)  # a product of 8 and 24 bits is rounded to fp32 and to the type
        assert torch.equal(got[i][:cu[-1]].cpu(), ref) and not got[i][cu[-1]:].any()
        assert torch.equal(by_slot[i].cpu(), ref)
    # a request whose row is not there has no rows; keys past the row's end neither
    bad = fa.read_quantized_kvcache(*c.args(DEV), cu_seqlens_k=i32([0, 3, 6]), total_k=6, cache_batch_idx=i32([99, -1]), dtype=out, **more)
    assert not bad[0].any() and not bad[1].any()
    far = fa.read_quantized_kvcache(*c.args(DEV), cu_seqlens_k=i32([2, 4, 3000]), total_k=3005, cache_batch_idx=i32([0, 0]), dtype=out, **more)
    x, _ = one(0, 0)
    assert not far[0][:2].any() and torch.equal(far[0][2:4].cpu(), x[:2].float().to(out))
    assert torch.equal(far[0][4:4 + lens[0]].cpu(), x.float().to(out)) and not far[0][4 + 3 * 144:].any()


def test_types_of_torch():
    """float4_e2m1fn_x2 and float8_e8m0fnu in place of their bytes."""
    print("case fp4 torch types", flush=True)
    g = torch.Generator().manual_seed(5)
    c = Cache4(g, [40, 20], 2, 64, 16)
    raw = c.args(DEV)
    typed = [t.view(torch.float4_e2m1fn_x2) for t in raw[:2]] + [t.view(torch.float8_e8m0fnu) for t in raw[2:]]
    q = torch.randn(2, 1, 4, 64, generator=g).to(torch.bfloat16).to(DEV)
    a = fa.flash_attn_with_quantized_kvcache(q, *raw, i32(c.lens), page_table=c.table.to(DEV))
    b = fa.flash_attn_with_quantized_kvcache(q, *typed, i32(c.lens), page_table=c.table.to(DEV))
    assert torch.equal(a, b)
    k = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    fa.append_quantized_kvcache(k, k, *typed, torch.tensor([17, 18], device=DEV))
    x, y = fa.read_quantized_kvcache(*typed, slot_mapping=torch.tensor([17, 18], device=DEV))
    assert x.dtype == torch.bfloat16 and torch.equal(x, y) and (x - k).abs().max() < k.abs().max() / 5


def test_streams_and_graph():
    """On a stream of its own, and captured: each replay appends, attends and reads what its inputs then hold."""
    print("case fp4 graph", flush=True)
    g = torch.Generator().manual_seed(6)
    Hk, H, D, page = 2, 8, 64, 16
    c = Cache4(g, [60, 33], Hk, D, page)
    dev = c.args(DEV)
    host = [t.clone() for t in (*c.codes, *c.scales)]
    table, lens = c.table.to(DEV), i32(c.lens)
    last = [c.pages[b][(n - 1) // page] * page + (n - 1) % page for b, n in enumerate(c.lens)]
    k, v = (torch.zeros(2, Hk, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(2, 1, H, D, dtype=torch.bfloat16, device=DEV)
    slots = torch.tensor(last, device=DEV)

    def step():
        fa.append_quantized_kvcache(k, v, *dev, slots)
        return (*fa.flash_attn_with_quantized_kvcache(q, *dev, lens, page_table=table, causal=True, return_softmax_lse=True),
                *fa.read_quantized_kvcache(*dev, slot_mapping=slots))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, rk, rv = step()
    for turn in range(3):
        x, y = (torch.randn(2, Hk, D, generator=g).to(torch.bfloat16) for _ in range(2))
        z = torch.randn(2, 1, H, D, generator=g).to(torch.bfloat16)
        k.copy_(x)
        v.copy_(y)
        q.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        fo.append(x, host[0], host[2], last)
        fo.append(y, host[1], host[3], last)
        same_cache(dev, host)
        c.codes, c.scales = host[:2], host[2:]
        for b in range(2):
            kk, vv, ok = c.rows(b, torch.bfloat16)
            check_attend4(out[b], lse[b], z[b], kk, vv, ok, torch.bfloat16, causal=True)
            assert torch.equal(rk[b].cpu().double(), kk[-1]) and torch.equal(rv[b].cpu().double(), vv[-1])
        eager = step()
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)


def test_serving_steps():
    """Requests come, decode, are taken back by a token and end over a pool that they share, q and k turned by their positions
    before the append; after every step the attention's result is that of the definitions run beside it."""
    print("case fp4 serving", flush=True)
    from oracle import fa_rotary_oracle as ro
    g, r = torch.Generator().manual_seed(31), random.Random(31)
    rows, width, page, Hk, H, D, rd, n = 6, 8, 16, 2, 8, 64, 32, 30
    st = [torch.zeros(n, page, Hk, D // 2, dtype=torch.uint8) for _ in range(2)] + \
         [torch.full((n, page, Hk, D // 32), 255, dtype=torch.uint8) for _ in range(2)]
    dev = [t.to(DEV) for t in st]
    how = dict(base=10000.0, scaling="by_parts", factor=4.0, original_length=32)
    cos, sin = fa.rotary_cos_sin(torch.arange(width * page, device=DEV), rd, attention_factor=1.1, **how)
    ref_cos, ref_sin = ro.table(range(width * page), rd, attention_factor=1.1, **how)
    assert (cos.cpu().double() - ref_cos).abs().max() < 2.0 ** -22 and (sin.cpu().double() - ref_sin).abs().max() < 2.0 ** -22
    table, free, num = [[0] * width for _ in range(rows)], list(range(n)), n
    t_dev, f_dev, num_dev = i32(table), i32(free), i32([num])
    lens = [0] * rows
    for turn in range(10):
        idx = sorted(r.sample(range(rows), r.randrange(2, rows + 1)))
        before = [lens[i] for i in idx]
        after = [r.randrange(1, 3 * page) if x == 0 else 0 if r.random() < 0.2 else x - 1 if r.random() < 0.15
                 else x + r.choice([1, 1, 1, 4]) for x in before]
        total = sum(max(y - x, 0) for x, y in zip(before, after))
        pad = total + 3  # a padded batch
        slots, cu, num_dev = fa.update_page_table(t_dev, i32(before), i32(after), f_dev, num_dev, page, pad,
                                                  cache_batch_idx=i32(idx))
        table, free, want, cu_want, num = qo.page_table_step(table, before, after, free, num, page, pad, idx=idx)
        k, v = (torch.randn(pad, Hk, D, generator=g).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(pad, H, D, generator=g).to(torch.bfloat16)
        qt, kt = fa.apply_rotary_emb(q.to(DEV), k.to(DEV), cos, sin, seqlen_offsets=i32(before), cu_seqlens=cu)
        fresh = [max(y - x, 0) for x, y in zip(before, after)]
        place = [x + j for x, m in zip(before, fresh) for j in range(m)]
        for got, x in ((qt, q), (kt, k)):
            ref = ro.turn(x[:total], cos.cpu()[place], sin.cpu()[place], True)
            assert torch.equal(got[total:].cpu(), x[total:])
            assert ((got[:total].cpu().double() - ref).abs() <= ref.abs() * 2.0 ** -8 + 2.0 ** -20).all()
        fa.append_quantized_kvcache(kt, v.to(DEV), *dev, slots)
        fo.append(kt.cpu(), st[0], st[2], want)
        fo.append(v, st[1], st[3], want)
        out, lse = fa.flash_attn_with_quantized_kvcache(qt, *dev, i32(after), page_table=t_dev, cache_batch_idx=i32(idx),
                                                        cu_seqlens_q=cu, max_seqlen_q=max(fresh + [1]), causal=True,
                                                        return_softmax_lse=True)
        assert slots.tolist() == want and cu.tolist() == cu_want and num_dev.item() == num
        same_cache(dev, st)
        at = 0
        for i, y, m in zip(idx, after, fresh):
            lens[i] = y
            if m:
                kk, ok = fo.rows_of(st[0], st[2], table[i], y)
                vv, _ = fo.rows_of(st[1], st[3], table[i], y)
                check_attend4(out[at:at + m], lse[:, at:at + m], qt[at:at + m].cpu(), kk, vv, ok, torch.bfloat16, causal=True)
            at += m


def test_refusals():
    """Wrong types, shapes and devices raise before anything is launched."""
    print("case fp4 refusals", flush=True)
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device=DEV)  # noqa: E731
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=DEV)  # noqa: E731
    kc, vc, ks, vs = u8(5, 32, 2, 32), u8(5, 32, 2, 32), u8(5, 32, 2, 2), u8(5, 32, 2, 2)
    good = dict(q=mk(2, 1, 8, 64), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, cache_seqlens=i32([0, 0]), page_table=i32([[0, 1], [2, 3]]))
    fa.flash_attn_with_quantized_kvcache(**good)
    for bad in (dict(q=mk(2, 1, 8, 64, dt=torch.float32)), dict(q=mk(2, 1, 8, 32)), dict(q=mk(2, 1, 7, 64)),
                dict(k_cache=u8(5, 32, 2, 64), v_cache=u8(5, 32, 2, 64)), dict(v_cache=vc.view(torch.int8)),
                dict(k_scale=ks.float(), v_scale=vs.float()), dict(k_scale=u8(5, 32, 2, 1), v_scale=u8(5, 32, 2, 1)),
                dict(k_scale=u8(5, 2, 2, 2), v_scale=u8(5, 2, 2, 2)), dict(k_scale=u8(5, 32, 2), v_scale=u8(5, 32, 2)),
                dict(k_cache=u8(5, 24, 2, 32), v_cache=u8(5, 24, 2, 32), k_scale=u8(5, 24, 2, 2), v_scale=u8(5, 24, 2, 2)),
                dict(q=mk(2, 1, 8, 48), k_cache=u8(5, 32, 2, 24), v_cache=u8(5, 32, 2, 24)),
                dict(k_scale=ks.cpu()), dict(k_scale=u8(5, 32, 2, 4)[..., ::2], v_scale=u8(5, 32, 2, 4)[..., ::2]),
                dict(cache_seqlens=mk(2, dt=torch.int64)), dict(softcap=-1.0)):
        with pytest.raises(RuntimeError):
            fa.flash_attn_with_quantized_kvcache(**dict(good, **bad))
    app = dict(k=mk(3, 2, 64), v=mk(3, 2, 64), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slot_mapping=mk(3, dt=torch.int64))
    for bad in (dict(k=mk(3, 2, 64, dt=torch.float32)), dict(v=mk(3, 2, 64, dt=torch.float16)), dict(k=mk(3, 1, 64), v=mk(3, 1, 64)),
                dict(slot_mapping=mk(3, dt=torch.int32)), dict(k=mk(3, 2, 32), v=mk(3, 2, 32)), dict(v_scale=vs.cpu())):
        with pytest.raises(RuntimeError):
            fa.append_quantized_kvcache(**dict(app, **bad))
    cache = (kc, vc, ks, vs)
    slots = mk(3, dt=torch.int64)
    for bad in (dict(), dict(slot_mapping=slots, cu_seqlens_k=i32([0, 3]), total_k=3), dict(slot_mapping=slots, dtype=torch.float64),
                dict(slot_mapping=slots.int()), dict(cu_seqlens_k=i32([0, 3])), dict(cu_seqlens_k=i32([0]), total_k=3),
                dict(cu_seqlens_k=i32([0, 1]).long(), total_k=1), dict(slot_mapping=slots, page_table=i32([[0]])),
                dict(cu_seqlens_k=i32([0, 1, 2]), total_k=2, page_table=i32([[0]])), dict(cu_seqlens_k=i32([0] * 7), total_k=2),
                dict(cu_seqlens_k=i32([0, 1]), total_k=-1), dict(cu_seqlens_k=i32([0, 1]), total_k=1, cache_batch_idx=i32([0, 0]))):
        with pytest.raises(RuntimeError):
            fa.read_quantized_kvcache(*cache, **bad)
