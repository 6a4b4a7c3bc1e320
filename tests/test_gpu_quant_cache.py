"""update_page_table and append_quantized_kvcache against their definitions (exactly: their results are whole
numbers, and codes whose scales are powers of two), and a run of serving steps with the attention behind them."""
import math
import random

import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_quant_oracle as qo
from tests._quant import CACHES, TYPES, check_attend, largest

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def i32(x):
    return torch.tensor(x, **I32)


def step(table, before, after, free, num_free, page, total, idx=None):
    """The operator on the same lists that the oracle takes."""
    t, f = i32(table), i32(free)
    slots, cu, left = fa.update_page_table(t, i32(before), i32(after), f, i32([num_free]), page, total,
                                           cache_batch_idx=None if idx is None else i32(idx))
    assert slots.dtype == torch.int64 and cu.dtype == torch.int32 and left.dtype == torch.int32
    return t.tolist(), f.tolist(), slots.tolist(), cu.tolist(), left.item()


def server(r, B, width, page, spare, done=0.2, extra_rows=0):
    """A page table in use and a step of it."""
    rows = B + extra_rows
    cap = width * page
    before = [r.choice([0, 1, page - 1, page, page + 1, cap - 1, cap, r.randrange(cap + 1)]) for _ in range(B)]
    before = [min(max(x, 0), cap) for x in before]
    after = [0 if r.random() < done else min(x + r.choice([0, 1, 1, 2, page, r.randrange(3 * page)]), cap)
             if r.random() < 0.8 else r.randrange(x + 1) for x in before]
    ids = list(range(sum(-(-x // page) for x in before) + spare))
    r.shuffle(ids)
    table = [[r.randrange(-3, 99) for _ in range(width)] for _ in range(rows)]
    idx = r.sample(range(rows), B) if extra_rows else None
    for b, x in enumerate(before):
        for j in range(-(-x // page)):
            table[idx[b] if idx else b][j] = ids.pop()
    free = ids + [-9] * (sum(-(-x // page) for x in before))
    total = sum(max(y - x, 0) for x, y in zip(before, after))
    return table, before, after, free, len(ids), page, total, idx


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 300, 1024, 1025, 3000, 4096, 4097])
@pytest.mark.parametrize("page", [1, 16, 48, 256])
def test_steps_of_a_server(B, page):
    print(f"case table {B} {page}", flush=True)
    r = random.Random(B * 1000 + page)
    for extra in (0, 3):
        a = server(r, B, 9, page, 8 * B, extra_rows=extra)
        assert step(*a) == qo.page_table_step(a[0], *a[1:7], idx=a[7])


@pytest.mark.parametrize("spare", [0, 1, 5])
def test_stack_runs_empty(spare):
    print(f"case empty stack {spare}", flush=True)
    r = random.Random(spare)
    for done in (0.0, 0.3):
        a = server(r, 100, 7, 8, spare, done=done)
        got = step(*a)
        assert got == qo.page_table_step(a[0], *a[1:7])
        # the next step: requests that got no page end, and no id below 0 comes onto the stack
        b = (got[0], a[2], [0] * 100, got[1], got[4], 8, 0)
        got = step(*b)
        assert got == qo.page_table_step(*b) and all(x >= 0 for x in got[1][:got[4]])


def test_lengths_out_of_range():
    """Negative lengths, lengths past the table, rows that are not in it, fewer slots than tokens, a count that is
    not one, a stack without room."""
    print("case lengths out of range", flush=True)
    table = [[1, 2, 3], [4, 5, 6], [7, 8, 9]]
    for args in (
        (table, [-5, 0, 12], [3, 30, 40], [20, 21, 22, 23, 24, 25], 6, 4, 80, None),
        (table, [12, 12, 0], [0, 100, 2], [20, 21, 22, 23, 24, 25], 2, 4, 100, None),
        (table, [12, 3, 0], [0, 5, 5], [20, 21, 22, 23, 24, 25], 5, 4, 20, [2, 17, -1]),
        (table, [0, 0, 0], [9, 9, 9], [20, 21, 22, 23, 24, 25], 9, 4, 5, None),
        (table, [0, 0, 8], [9, 9, 0], [20, 21, 22, 23, 24, 25], -4, 4, 18, None),
        (table, [12, 12, 12], [0, 0, 0], [20, 21], 1, 4, 0, None),
        (table, [12, 12, 12], [0, 0, 12], [], 0, 4, 3, None),
        ([[], []], [0, 3], [4, 2], [5], 1, 4, 4, None),
    ):
        assert step(*args) == qo.page_table_step(args[0], *args[1:7], idx=args[7])


def test_a_step_taken_twice_is_one_step():
    print("case step twice", flush=True)
    a = server(random.Random(5), 200, 6, 16, 500)
    t, f = i32(a[0]), i32(a[3])
    args = (t, i32(a[1]), i32(a[2]), f, i32([a[4]]), a[5], a[6])
    one = [x.tolist() for x in fa.update_page_table(*args)] + [t.tolist(), f.tolist()]
    two = [x.tolist() for x in fa.update_page_table(*args)] + [t.tolist(), f.tolist()]
    assert one == two


def test_long_prompts():
    print("case long prompts", flush=True)
    r = random.Random(6)
    before = [r.randrange(20) for _ in range(40)]
    after = [x + r.randrange(1, 20000) for x in before]
    pages = sum(-(-y // 16) for y in after)
    ids = list(range(pages))
    r.shuffle(ids)
    table = [[0] * 1300 for _ in range(40)]
    for b in range(40):
        for j in range(-(-before[b] // 16)):
            table[b][j] = ids.pop()
    total = sum(after) - sum(before)
    a = (table, before, after, ids + [0] * 40, len(ids), 16, total + 100)
    assert step(*a) == qo.page_table_step(*a)
    # all of them end
    got = step(*a)
    b = (got[0], after, [0] * 40, got[1], got[4], 16, 0)
    assert step(*b) == qo.page_table_step(*b)


def test_strided_table_and_graph():
    print("case table graph", flush=True)
    big = torch.full((5, 40), -7, **I32)
    table = big[:, 3:12]
    a = server(random.Random(7), 5, 9, 16, 60, done=0.0)
    table.copy_(i32(a[0]))
    before, after, free, num = i32(a[1]), i32(a[2]), i32(a[3]), i32([a[4]])
    call = lambda: fa.update_page_table(table, before, after, free, num, 16, 200)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, cu, left = call()
    for seed in range(4):
        a = server(random.Random(seed + 70), 5, 9, 16, 60)
        for t, x in ((table, a[0]), (before, a[1]), (after, a[2]), (num, [a[4]])):
            t.copy_(i32(x))
        free[:len(a[3])] = i32(a[3])[:free.numel()]
        was = free.tolist()
        graph.replay()
        torch.cuda.synchronize()
        want = qo.page_table_step(a[0], a[1], a[2], was, a[4], 16, 200)
        assert (table.tolist(), free.tolist(), slots.tolist(), cu.tolist(), left.item()) == want
        assert (big[:, :3] == -7).all() and (big[:, 12:] == -7).all()


# ---- append -------------------------------------------------------------------------------------


def filled(g, n, page, Hk, D, dt, block):
    """A cache as earlier appends left it: any codes, scales that are powers of two."""
    top = qo.CODE_MAX[dt]
    out = []
    for _ in range(2):
        x = (torch.randn(n, page, Hk, D, generator=g) * top / 3.5).clamp(-top, top)
        out.append((x.round() if dt == torch.int8 else x).to(dt))
    for _ in range(2):
        out.append(2.0 ** torch.randint(-12, 2, (n, page // block, Hk), generator=g).float())
    return out


def check_append(k, v, st, slots, slots_dev=None):
    """The call on the GPU against the definition, bit for bit (a NaN has two codes)."""
    want = [t.clone() for t in st]
    dev = [t.to(DEV) for t in st]
    fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), *dev,
                                torch.tensor(slots, dtype=torch.int64, device=DEV) if slots_dev is None else slots_dev)
    for i, x in enumerate((k, v)):
        qo.append(x, want[i], want[2 + i], slots)
        assert torch.equal(dev[2 + i].cpu(), want[2 + i]), "scales differ"
        a, b = dev[i].cpu().view(torch.uint8).int(), want[i].view(torch.uint8).int()
        if want[i].dtype != torch.int8:
            a, b = (torch.where(t & 0x7f == 0x7f, 0x7f, t) for t in (a, b))
            a, b = (torch.where(t == 0x80, 0, t) for t in (a, b))  # and zero a sign
        assert torch.equal(a, b), "codes differ"


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (64, 64), (256, 128)])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_append_runs(dt, cache, page, block):
    """Runs that begin a block, continue one, end one, cross pages; rows without a slot between them."""
    print(f"case append {dt} {cache} {page}/{block}", flush=True)
    g = torch.Generator().manual_seed(20)
    r = random.Random(20)
    n = 12
    st = filled(g, n, page, 3, 64, CACHES[cache], block)
    pages = r.sample(range(n), n)
    slots = []
    for first, count in ((0, 1), (5, 1), (0, page), (block - 1, 2 if page > block else 1), (3, page - 3), (page - 1, 1)):
        p = pages.pop()
        slots += [p * page + first + i for i in range(count)]
    p, p2 = pages.pop(), pages.pop()
    slots += [p * page + page - 2, p * page + page - 1, p2 * page, p2 * page + 1]
    slots += [-1, -1, n * page, n * page + 5, -(1 << 40), 1 << 40]
    p = pages.pop()
    slots += [p * page + 7, p * page + 8]
    k, v = ((torch.randn(len(slots), 3, 64, generator=g) * 2.0 ** torch.randint(-6, 4, (len(slots), 3, 1), generator=g))
            .to(TYPES[dt]) for _ in range(2))
    check_append(k, v, st, slots)


@pytest.mark.parametrize("D", [16, 48, 80, 128, 192, 256])
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_append_head_dims(D, cache):
    print(f"case append head dim {D} {cache}", flush=True)
    g = torch.Generator().manual_seed(21)
    st = filled(g, 3, 64, 5, D, CACHES[cache], 32)
    slots = [64 + i for i in range(3, 64)] + [20, 21]
    k, v = (torch.randn(len(slots), 5, D, generator=g).to(torch.bfloat16) for _ in range(2))
    check_append(k, v, st, slots)


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_append_extremes(dt, cache):
    """Zeros, subnormals, the largest values, infinities and NaN; every 16-bit value; values at rounding ties."""
    print(f"case append extremes {dt} {cache}", flush=True)
    g = torch.Generator().manual_seed(22)
    t = TYPES[dt]
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    rows = [torch.zeros(64), torch.full((64,), big), torch.full((64,), -tiny / 4), torch.full((64,), math.inf),
            torch.full((64,), math.nan), torch.full((64,), -0.0)]
    for x in (math.inf, -math.inf, math.nan, big, tiny):
        y = torch.randn(64, generator=g)
        y[7] = x
        rows.append(y)
    rows.append(torch.arange(64) + 0.5)
    rows.append((torch.arange(64) * 2 + 1) * 2.0 ** -10)
    every = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(t).float().view(-1, 64)
    x = torch.stack(rows).to(t)
    x = torch.cat([x, every.to(t)])[:, None]
    n = x.shape[0]
    for begun in (False, True):
        st = filled(g, n, 16, 1, 64, CACHES[cache], 16)
        check_append(x, x.flip(0), st, [i * 16 + (5 if begun else 0) for i in range(n)])


def test_append_into_scales_of_any_value():
    """Blocks that were calibrated: a scale that is no power of two stays where it is the larger."""
    print("case append odd scales", flush=True)
    g = torch.Generator().manual_seed(23)
    for dt in (torch.int8, torch.float8_e4m3fn):
        st = filled(g, 8, 16, 2, 32, dt, 16)
        for s in st[2:]:
            s.copy_(torch.rand(s.shape, generator=g) + 0.5)
        k, v = (torch.randn(8, 2, 32, generator=g).to(torch.bfloat16) for _ in range(2))
        # x / s is rounded to 24 bits before it becomes a code: another code than from 64 bits needs a quotient
        # within 2^-25 of a tie, which these inputs do not have
        check_append(k, v, st, [i * 16 + 3 for i in range(8)])


def test_append_strides():
    print("case append strides", flush=True)
    g = torch.Generator().manual_seed(24)
    st = filled(g, 4, 32, 2, 64, torch.int8, 16)
    qkv = torch.randn(40, 8, 64, generator=g).to(torch.float16)
    k, v = qkv[:, 4:6], qkv[:, 6:8]
    slots = list(range(5, 45))
    want = [t.clone() for t in st]
    qo.append(k, want[0], want[2], slots)
    qo.append(v, want[1], want[3], slots)
    q = qkv.to(DEV)
    odd = torch.empty(40, 2, 65, dtype=torch.float16, device=DEV)[:, :, 1:]  # rows that are not 16-byte aligned
    odd.copy_(q[:, 4:6])
    both = torch.zeros(4, 2, 32, 2, 64, dtype=torch.int8, device=DEV)  # page, head, row, k / v, dim
    views = [both[:, :, :, i].transpose(1, 2) for i in (0, 1)]
    scales = [t.to(DEV).permute(2, 1, 0).contiguous().permute(2, 1, 0) for t in st[2:]]
    for kk in (q[:, 4:6], odd):
        for view, t in zip(views, st):
            view.copy_(t.to(DEV))
        for s, t in zip(scales, st[2:]):
            s.copy_(t.to(DEV))
        fa.append_quantized_kvcache(kk, q[:, 6:8], *views, *scales, torch.tensor(slots, device=DEV))
        for view, s, w, ws in zip(views, scales, want[:2], want[2:]):
            assert torch.equal(view.cpu(), w) and torch.equal(s.cpu(), ws)


def test_append_prompts():
    """Blocks of every kind at once, as long prompts fill them."""
    print("case append prompts", flush=True)
    g = torch.Generator().manual_seed(25)
    for cache, page, block, D in (("int8", 256, 256, 64), ("e4m3", 128, 64, 128), ("int8", 64, 16, 256)):
        n = 24
        st = filled(g, n, page, 2, D, CACHES[cache], block)
        slots = list(range(page + 3, 9 * page + 11)) + list(range(12 * page, 15 * page - 1)) + [20 * page + page - 1]
        k, v = (torch.randn(len(slots), 2, D, generator=g).to(torch.bfloat16) for _ in range(2))
        check_append(k, v, st, slots)


def test_append_offsets_past_32_bits():
    print("case append past 32 bits", flush=True)
    g = torch.Generator().manual_seed(26)
    n, P, Hk, D = 36000, 128, 8, 128
    k8, v8 = (torch.zeros(n, P, Hk, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(n, 1, Hk, device=DEV) for _ in range(2))
    slots = [(n - 1) * P + i for i in range(P)] + [0]
    k, v = (torch.randn(len(slots), Hk, D, generator=g).to(torch.bfloat16) for _ in range(2))
    fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), k8, v8, ks, vs, torch.tensor(slots, device=DEV))
    for x, c, s in ((k, k8, ks), (v, v8, vs)):
        small, sc = torch.zeros(2, P, Hk, D, dtype=torch.int8), torch.zeros(2, 1, Hk)
        qo.append(x, small, sc, [P + i for i in range(P)] + [0])
        assert torch.equal(c[n - 1].cpu(), small[1]) and torch.equal(c[0].cpu(), small[0])
        assert torch.equal(s[n - 1].cpu(), sc[1]) and torch.equal(s[0].cpu(), sc[0])


def test_append_graph():
    print("case append graph", flush=True)
    g = torch.Generator().manual_seed(27)
    st = filled(g, 4, 32, 2, 64, torch.int8, 16)
    dev = [t.to(DEV) for t in st]
    k, v = (torch.zeros(6, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots = torch.full((6,), -1, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.append_quantized_kvcache(k, v, *dev, slots)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(dev, st))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa.append_quantized_kvcache(k, v, *dev, slots)
    for at in ([0, 1, 2, 40, 41, -1], [3, 4, 42, 43, 96, 97], [-1] * 6, [5, 6, 7, 8, 9, 10]):
        x, y = (torch.randn(6, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
        k.copy_(x)
        v.copy_(y)
        slots.copy_(torch.tensor(at))
        graph.replay()
        torch.cuda.synchronize()
        qo.append(x, st[0], st[2], at)
        qo.append(y, st[1], st[3], at)
        assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(dev, st))


def test_refusals():
    """Wrong types, shapes and devices raise before anything is launched."""
    print("case refusals", flush=True)
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(s, device=DEV).to(dt)  # noqa: E731
    f32, i8, i64 = torch.float32, torch.int8, torch.int64
    good = dict(q=mk(2, 1, 8, 64), k_cache=mk(5, 32, 2, 64, dt=i8), v_cache=mk(5, 32, 2, 64, dt=i8),
                k_scale=mk(5, 2, 2, dt=f32), v_scale=mk(5, 2, 2, dt=f32), cache_seqlens=mk(2, dt=torch.int32),
                page_table=mk(2, 2, dt=torch.int32))
    fa.flash_attn_with_quantized_kvcache(**good)
    for bad in (dict(q=mk(2, 1, 8, 64, dt=f32)), dict(q=mk(2, 8, 64)), dict(q=mk(2, 1, 7, 64)), dict(q=mk(2, 1, 8, 32)),
                dict(k_cache=mk(5, 32, 2, 64)), dict(v_cache=mk(5, 32, 2, 64, dt=torch.float8_e4m3fn)),
                dict(v_cache=mk(5, 16, 2, 64, dt=i8)), dict(k_scale=mk(5, 2, 2)), dict(k_scale=mk(5, 2, 1, dt=f32)),
                dict(k_scale=mk(5, 3, 2, dt=f32), v_scale=mk(5, 3, 2, dt=f32)),
                dict(k_scale=mk(5, 4, 2, dt=f32), v_scale=mk(5, 4, 2, dt=f32)), dict(cache_seqlens=mk(2, dt=i64)),
                dict(cache_seqlens=mk(3, dt=torch.int32)), dict(page_table=mk(1, 2, dt=torch.int32)),
                dict(page_table=mk(2, 2, dt=i64)), dict(page_table=good["page_table"].cpu()), dict(k_cache=good["k_cache"].cpu()),
                dict(cache_batch_idx=mk(3, dt=torch.int32)), dict(softcap=-1.0),
                dict(cu_seqlens_q=mk(3, dt=torch.int32), max_seqlen_q=1),
                dict(q=mk(2, 8, 64), cu_seqlens_q=mk(3, dt=i64), max_seqlen_q=1)):
        with pytest.raises(RuntimeError):
            fa.flash_attn_with_quantized_kvcache(**dict(good, **bad))
    app = dict(k=mk(3, 2, 64), v=mk(3, 2, 64), k_cache=good["k_cache"], v_cache=good["v_cache"], k_scale=good["k_scale"],
               v_scale=good["v_scale"], slot_mapping=mk(3, dt=i64))
    for bad in (dict(k=mk(3, 2, 64, dt=f32)), dict(v=mk(3, 2, 64, dt=torch.float16)), dict(v=mk(2, 2, 64)), dict(k=mk(3, 1, 64), v=mk(3, 1, 64)),
                dict(slot_mapping=mk(3, dt=torch.int32)), dict(slot_mapping=mk(2, dt=i64)), dict(v_scale=good["v_scale"].cpu()),
                dict(k=mk(3, 2, 32), v=mk(3, 2, 32)), dict(slot_mapping=mk(3, dt=i64).cpu())):
        with pytest.raises(RuntimeError):
            fa.append_quantized_kvcache(**dict(app, **bad))
    i = lambda *s: mk(*s, dt=torch.int32)  # noqa: E731
    up = dict(page_table=i(4, 3), cache_seqlens=i(4), new_seqlens=i(4), free_pages=i(5), num_free=i(1), page_size=16, total_new=2)
    for bad in (dict(page_table=mk(4, 3, dt=i64)), dict(page_table=i(3, 3)), dict(page_table=i(4, 6)[:, ::2]), dict(new_seqlens=i(3)),
                dict(num_free=i(2)), dict(free_pages=mk(5, dt=i64)), dict(page_size=0), dict(total_new=-1),
                dict(cache_batch_idx=i(2)), dict(cache_seqlens=i(0), new_seqlens=i(0)), dict(free_pages=i(5).cpu())):
        with pytest.raises(RuntimeError):
            fa.update_page_table(**dict(up, **bad))


# ---- together -----------------------------------------------------------------------------------


@pytest.mark.parametrize("cache,page,block", [("int8", 32, 16), ("e4m3", 64, 64)])
def test_serving_steps(cache, page, block):
    """Requests come, decode, are taken back by a token and end over a pool that they share; after every step the
    attention's result is that of the definitions run beside it."""
    print(f"case serving {cache}", flush=True)
    g, r = torch.Generator().manual_seed(30), random.Random(30)
    rows, width, Hk, H, D, n = 6, 8, 2, 8, 128, 30
    dt = CACHES[cache]
    st = [torch.zeros(n, page, Hk, D).to(dt) for _ in range(2)] + [torch.full((n, page // block, Hk), math.nan) for _ in range(2)]
    dev = [t.to(DEV) for t in st]
    table, free, num = [[0] * width for _ in range(rows)], list(range(n)), n
    t_dev, f_dev, num_dev = i32(table), i32(free), i32([num])
    lens = [0] * rows
    for turn in range(12):
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
        fa.append_quantized_kvcache(k.to(DEV), v.to(DEV), *dev, slots)
        qo.append(k, st[0], st[2], want)
        qo.append(v, st[1], st[3], want)
        q = torch.randn(pad, H, D, generator=g).to(torch.bfloat16)
        fresh = [max(y - x, 0) for x, y in zip(before, after)]
        out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), *dev, i32(after), page_table=t_dev,
                                                        cache_batch_idx=i32(idx), cu_seqlens_q=cu,
                                                        max_seqlen_q=max(fresh + [1]), causal=True, return_softmax_lse=True)
        assert slots.tolist() == want and cu.tolist() == cu_want and num_dev.item() == num
        assert t_dev.tolist() == table and f_dev.tolist() == free
        for i, y in zip(idx, after):
            lens[i] = y
        at = 0
        for i, y, m in zip(idx, after, fresh):
            if m:
                kk, ok = qo.rows_of(st[0], st[2], table[i], y)
                vv, _ = qo.rows_of(st[1], st[3], table[i], y)
                check_attend(out[at:at + m], lse[:, at:at + m], q[at:at + m], kk, vv, ok, largest(st[1], st[3]),
                             torch.bfloat16, causal=True)
            at += m
