"""rotary_cos_sin and apply_rotary_emb against oracle/fa_rotary_oracle.py: tables, rotation, gradients."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_rotary_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


HOWS = [dict(), dict(scaling="linear", factor=2.5), dict(scaling="ntk", factor=16.0, base=500000.0),
        dict(scaling="by_parts", factor=8.0, original_length=4096, low=1.0, high=4.0)]


@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("rd", [16, 48, 128, 256])
@pytest.mark.parametrize("table", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("wide", [False, True])
def test_table(how, rd, table, wide):
    """An angle is a product of two 64-bit numbers of 2^-53 each, so off by p f 2^-51 at most (host and oracle both
    round, and the turns taken out); sine and cosine of it are good to 2 steps of fp32 (2^-22), and the
    product by attention_factor and the rounding to the type half a step each. All are relative to the value except the
    angle's error and the 2^-24 that a turn's rest, rounded to fp32, is off at most by half a turn (times pi)."""
    print(f"case table {how} {rd} {table}", flush=True)
    dt, att = TYPES[table], 1.25
    pos = [0, 1, 2, 3, 17, 1023, 4096, 65537, 131071, 1048575, 16777217, 2 ** 31 - 1, -1, -77] + ([2 ** 33 + 5] if wide else [])
    t = torch.tensor(pos, dtype=torch.int64 if wide else torch.int32, device=DEV)
    got = fa.rotary_cos_sin(t, rd, attention_factor=att, dtype=dt, **how)
    f = torch.tensor(ro.frequencies(rd, **how), dtype=torch.float64)
    p = torch.tensor(pos, dtype=torch.float64)[:, None]
    for y, ref in zip(got, ro.table(pos, rd, attention_factor=att, **how)):
        assert y.dtype == dt and y.shape == ref.shape
        off = att * ((p * f).abs() * 2.0 ** -50 + math.pi * 2.0 ** -24) + ref.abs() * (2.0 ** -22 + 2.0 ** -24)
        half = torch.finfo(dt).eps / 2
        bound = off + ref.abs() * half + torch.finfo(dt).smallest_normal * half
        worst = ((y.cpu().double() - ref).abs() / bound).max().item()
        assert worst <= 1, worst


def test_table_sizes():
    """No positions, one, and so many that a workgroup ends inside a row; slices that are not contiguous."""
    print("case table sizes", flush=True)
    for n in (0, 1, 5, 1000):
        c, s = fa.rotary_cos_sin(torch.arange(n, device=DEV), 48)
        assert c.shape == s.shape == (n, 24)
        if n:
            ref = ro.table(range(n), 48)
            assert (c.cpu().double() - ref[0]).abs().max() < 2.0 ** -20 and (s.cpu().double() - ref[1]).abs().max() < 2.0 ** -20
    a, _ = fa.rotary_cos_sin(torch.arange(40, device=DEV)[::2], 32)
    b, _ = fa.rotary_cos_sin(torch.arange(0, 40, 2, device=DEV), 32)
    assert torch.equal(a, b)


def tables(n, rd, dt):
    cos, sin = ro.table(range(n), rd)
    return cos.to(dt).to(DEV), sin.to(dt).to(DEV)


def check(got, x, cos, sin, place, inter, dt, sign=1.0):
    """Each product is rounded to fp32 and their sum to the type: (|x1 c| + |x2 s|) 2^-23 and half a step."""
    c, s = cos.cpu().double()[place], sign * sin.cpu().double()[place]
    ref = ro.turn(x, c, s, inter)
    size = ro.turn(x.abs(), c.abs(), -s.abs(), inter).abs().maximum(ro.turn(x.abs(), c.abs(), s.abs(), inter).abs())
    half = torch.finfo(dt).eps / 2
    bound = size * 2.0 ** -23 + ref.abs() * half * (1 + 2.0 ** -10) + torch.finfo(dt).smallest_normal * half
    assert ((got.detach().cpu().double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("table", ["fp32", "same"])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("B,S,H,Hk,D,rd", [(1, 1, 1, 1, 16, 16), (2, 7, 4, 2, 64, 64), (3, 5, 3, 1, 80, 48), (1, 33, 8, 8, 256, 256),
                                           (2, 3, 5, 0, 264, 128)])
def test_dense(dtype, table, inter, B, S, H, Hk, D, rd):
    print(f"case rotate dense {dtype} {table} {inter} {B} {S} {H} {Hk} {D} {rd}", flush=True)
    g = torch.Generator().manual_seed(D + S)
    dt = TYPES[dtype]
    cos, sin = tables(60, rd, dt if table == "same" else torch.float32)
    q = torch.randn(B, S, H, D, generator=g).to(dt)
    k = torch.randn(B, S, Hk, D, generator=g).to(dt) if Hk else None
    dq, dk = (None if x is None else torch.randn(x.shape, generator=g).to(dt) for x in (q, k))
    starts = torch.randint(0, 20, (B,), generator=g)
    pos = torch.randint(0, 60, (B, S), generator=g)
    for how, place in ((dict(), torch.arange(S).expand(B, S)), (dict(seqlen_offsets=9), 9 + torch.arange(S).expand(B, S)),
                       (dict(seqlen_offsets=starts.int().to(DEV)), starts[:, None] + torch.arange(S)),
                       (dict(positions=pos.to(DEV)), pos), (dict(positions=pos.int().t().contiguous().t().to(DEV)), pos)):
        x, y = (None if t is None else t.to(DEV).requires_grad_() for t in (q, k))
        out = fa.apply_rotary_emb(x, y, cos, sin, rotary_interleaved=inter, **how)
        pairs = [(out, q, x, dq)] if k is None else [(out[0], q, x, dq), (out[1], k, y, dk)]
        grads = torch.autograd.grad([p[0] for p in pairs], [p[2] for p in pairs], [p[3].to(DEV) for p in pairs])
        for (got, src, _, d), gr in zip(pairs, grads):
            assert got.dtype == dt and got.shape == src.shape
            check(got, src, cos, sin, place, inter, dt)
            check(gr, d, cos, sin, place, inter, dt, sign=-1.0)
            assert torch.equal(got[..., rd:].cpu(), src[..., rd:]) and torch.equal(gr[..., rd:].cpu(), d[..., rd:])
        # in place: the same bits, of views into a larger tensor too, whose rest stays
        heads = H + Hk
        both = torch.randn(B, S, heads + 1, D, generator=g).to(dt)
        both[:, :, :H] = q
        if k is not None:
            both[:, :, H:heads] = k
        z = both.to(DEV)
        fa.apply_rotary_emb(z[:, :, :H], z[:, :, H:heads] if k is not None else None, cos, sin, rotary_interleaved=inter, inplace=True, **how)
        assert torch.equal(z[:, :, :H], pairs[0][0]) and torch.equal(z[:, :, heads:].cpu(), both[:, :, heads:])
        if k is not None:
            assert torch.equal(z[:, :, H:heads], pairs[1][0])


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("lens", [[1], [5, 0, 12, 1, 0], [3] * 40])
def test_ragged(inter, lens):
    """Sequences one behind the other; rows before the first and behind the last stay, gradients too."""
    print(f"case rotate ragged {inter} {len(lens)}", flush=True)
    g = torch.Generator().manual_seed(len(lens))
    dt, H, Hk, D, rd = torch.bfloat16, 4, 2, 48, 32
    cos, sin = tables(30, rd, torch.float32)
    cu = [2]
    for n in lens:
        cu.append(cu[-1] + n)
    T = cu[-1] + 4
    q, k = (torch.randn(T, h, D, generator=g).to(dt) for h in (H, Hk))
    starts = torch.randint(0, 15, (len(lens),), generator=g)
    place = torch.tensor([s + i for s, n in zip(starts.tolist(), lens) for i in range(n)])
    x, y = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    a, b = fa.apply_rotary_emb(x, y, cos, sin, seqlen_offsets=starts.int().to(DEV), cu_seqlens=i32(cu), rotary_interleaved=inter)
    ga, gb = torch.autograd.grad((a, b), (x, y), (x.detach(), y.detach()))
    live = slice(cu[0], cu[-1])
    for got, src, sign in ((a, q, 1.0), (b, k, 1.0), (ga, q, -1.0), (gb, k, -1.0)):
        check(got[live], src[live], cos, sin, place, inter, dt, sign)
        assert torch.equal(got[:cu[0]].cpu(), src[:cu[0]]) and torch.equal(got[cu[-1]:].cpu(), src[cu[-1]:])
    z = q.to(DEV)
    fa.apply_rotary_emb(z, None, cos, sin, seqlen_offsets=starts.int().to(DEV), cu_seqlens=i32(cu), rotary_interleaved=inter, inplace=True)
    assert torch.equal(z, a)


def test_positions_outside_the_tables():
    """Take the nearest row."""
    print("case rotate outside", flush=True)
    g = torch.Generator().manual_seed(8)
    cos, sin = tables(9, 16, torch.float32)
    q = torch.randn(6, 2, 16, generator=g).to(torch.float16)
    pos = torch.tensor([-1, -2 ** 40, 9, 2 ** 40, 8, 0])
    got = fa.apply_rotary_emb(q.to(DEV), None, cos, sin, positions=pos.to(DEV))
    check(got, q, cos, sin, torch.tensor([0, 0, 8, 8, 8, 0]), True, torch.float16)
    got = fa.apply_rotary_emb(q.to(DEV), None, cos, sin, seqlen_offsets=-2 ** 40)
    check(got, q, cos, sin, torch.zeros(6, dtype=torch.long), True, torch.float16)


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_same_bits_as_kvcache(inter, dtype):
    """The rows that flash_attn_with_kvcache appends with the same tables."""
    print(f"case rotate kvcache {inter} {dtype}", flush=True)
    g = torch.Generator().manual_seed(9)
    dt, B, S, H, Hk, D, rd = TYPES[dtype], 2, 5, 4, 2, 64, 32
    cos, sin = tables(80, rd, dt)
    q, k, v = (torch.randn(B, S, h, D, generator=g).to(dt).to(DEV) for h in (H, Hk, Hk))
    kc, vc = (torch.zeros(B, 64, Hk, D, dtype=dt, device=DEV) for _ in range(2))
    lens = i32([11, 40])
    out = fa.flash_attn_with_kvcache(q, kc, vc, k, v, rotary_cos=cos, rotary_sin=sin, cache_seqlens=lens, causal=True, rotary_interleaved=inter)
    qt, kt = fa.apply_rotary_emb(q, k, cos, sin, seqlen_offsets=lens, rotary_interleaved=inter)
    for b, n in enumerate([11, 40]):
        assert torch.equal(kc[b, n:n + S], kt[b])
    kc[:, 60:] = 0
    again = fa.flash_attn_with_kvcache(qt, kc, vc, cache_seqlens=lens + S, causal=True)
    assert (again.float() - out.float()).abs().max() < 2.0 ** -6


def test_training_step():
    """Attention over turned rows: gradients of q, k, v against those of the formula in 64 bits, and against differences."""
    print("case rotate training", flush=True)
    g = torch.Generator().manual_seed(10)
    dt, B, S, H, Hk, D, rd = torch.float16, 1, 24, 2, 1, 64, 32
    cos, sin = tables(S, rd, torch.float32)
    rows = [torch.randn(B, S, h, D, generator=g).to(dt) for h in (H, Hk, Hk)]
    w = torch.randn(B, S, H, D, generator=g).to(dt)
    leaves = [t.to(DEV).requires_grad_() for t in rows]
    q, k = fa.apply_rotary_emb(leaves[0], leaves[1], cos, sin)
    out = fa.flash_attn_func(q, k, leaves[2], causal=True)
    got = torch.autograd.grad(out, leaves, w.to(DEV))

    def loss(q, k, v):
        c, s = cos.cpu().double()[None], sin.cpu().double()[None]

        def turn(x):
            a, b = x[..., 0:rd:2], x[..., 1:rd:2]
            z = torch.stack((a * c[:, :, None] - b * s[:, :, None], b * c[:, :, None] + a * s[:, :, None]), -1).flatten(-2)
            return torch.cat((z, x[..., rd:]), -1)

        q, k = turn(q), turn(k).repeat_interleave(H // Hk, 2)
        x = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
        x = x.masked_fill(torch.ones(S, S).triu(1).bool(), -math.inf)
        return (torch.einsum("bhij,bjhd->bihd", x.softmax(-1), v.repeat_interleave(H // Hk, 2)) * w.double()).sum()

    ref = [t.double().requires_grad_() for t in rows]
    want = torch.autograd.grad(loss(*ref), ref)
    for a, b in zip(got, want):
        # 16-bit operands at four roundings of half a step each, sums over S and H rows: 8 of them at the size of the largest
        assert (a.cpu().double() - b).abs().max() <= 8 * 2.0 ** -11 * b.abs().max()
    with torch.no_grad():  # the formula's own gradients against differences: third derivatives times 1e-10, roundings over 1e-5
        for i in range(3):
            d = torch.randn(rows[i].shape, generator=g).double()
            up, down = ([t.double() + (e * d if j == i else 0) for j, t in enumerate(rows)] for e in (1e-5, -1e-5))
            slope = (loss(*up) - loss(*down)).item() / 2e-5
            assert abs((want[i] * d).sum().item() - slope) <= 1e-6 * (want[i].abs() * d.abs()).sum().item()


def test_gradients_of_one_and_broadcast():
    """Gradients that only q or only k asks for; incoming ones without memory of their own; leaves turned in place."""
    print("case rotate grads", flush=True)
    g = torch.Generator().manual_seed(11)
    cos, sin = tables(8, 32, torch.float32)
    q, k = (torch.randn(2, 8, h, 32, generator=g).to(torch.bfloat16).to(DEV) for h in (3, 1))
    place = torch.arange(8).expand(2, 8)
    for need_q, need_k in ((True, False), (False, True), (True, True)):
        x, y = q.clone().requires_grad_(need_q), k.clone().requires_grad_(need_k)
        a, b = fa.apply_rotary_emb(x, y, cos, sin)
        (a.sum() + b.sum()).backward()  # the incoming gradient is one number, expanded
        for leaf, need in ((x, need_q), (y, need_k)):
            assert (leaf.grad is not None) == need
            if need:
                check(leaf.grad, torch.ones(leaf.shape), cos, sin, place, True, torch.bfloat16, -1.0)
    x = q.clone().requires_grad_()
    a, _ = fa.apply_rotary_emb(x, k, cos, sin)  # only the first result is used
    a.backward(q)
    check(x.grad, q.cpu(), cos, sin, place, True, torch.bfloat16, -1.0)
    x = q.clone().requires_grad_()
    y = x * 1.0
    z = fa.apply_rotary_emb(y, None, cos, sin, inplace=True)
    assert z is y or z.data_ptr() == y.data_ptr()
    z.backward(q)
    check(x.grad, q.cpu(), cos, sin, place, True, torch.bfloat16, -1.0)
    with pytest.raises(RuntimeError):
        fa.apply_rotary_emb(q.clone().requires_grad_(), None, cos, sin, inplace=True)  # a leaf


def test_second_gradients():
    """The gradient of a gradient: the rotation again, of q and k and of one alone."""
    print("case rotate second gradients", flush=True)
    g = torch.Generator().manual_seed(14)
    cos, sin = tables(8, 32, torch.float32)
    place = torch.arange(8).expand(2, 8)
    for both in (True, False):
        x, dx, w = (torch.randn(2, 8, 3, 32, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3))
        x.requires_grad_()
        dx.requires_grad_()
        out = fa.apply_rotary_emb(x, x * 2 if both else None, cos, sin)
        (first,) = torch.autograd.grad(out[0] if both else out, x, dx, create_graph=True)
        check(first, dx.detach().cpu(), cos, sin, place, True, torch.bfloat16, -1.0)
        (second,) = torch.autograd.grad(first, dx, w)
        check(second, w.cpu(), cos, sin, place, True, torch.bfloat16)


def test_in_place_on_parts_of_a_projection():
    """q and k out of one projection, turned where they lie: right gradients, or a refusal by autograd."""
    print("case rotate projection", flush=True)
    g = torch.Generator().manual_seed(15)
    cos, sin = tables(8, 32, torch.float32)
    place = torch.arange(8).expand(2, 8)
    leaf = torch.randn(2, 8, 6, 32, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()
    d = torch.randn(2, 8, 6, 32, generator=g).to(torch.bfloat16)
    try:
        qkv = leaf * 1.0
        q, k = fa.apply_rotary_emb(qkv[:, :, :3], qkv[:, :, 3:5], cos, sin, inplace=True)
        (grad,) = torch.autograd.grad((q, k), leaf, (d[:, :, :3].to(DEV), d[:, :, 3:5].to(DEV)))
    except RuntimeError as e:
        assert "view" in str(e)
    else:
        check(grad[:, :, :5], d[:, :, :5], cos, sin, place, True, torch.bfloat16, -1.0)
    qkv = leaf.detach().clone()
    q, k = fa.apply_rotary_emb(qkv[:, :, :3], qkv[:, :, 3:5], cos, sin, inplace=True)
    check(qkv[:, :, :5], leaf.detach().cpu()[:, :, :5], cos, sin, place, True, torch.bfloat16)
    assert torch.equal(qkv[:, :, 5], leaf[:, :, 5]) and q.data_ptr() == qkv.data_ptr()


def test_captured_backward():
    """Forward and backward in one graph, leaves and gradients in place, replayed with other values."""
    print("case rotate captured backward", flush=True)
    g = torch.Generator().manual_seed(16)
    cos, sin = tables(8, 32, torch.float32)
    place = torch.arange(8)
    q, k = (torch.zeros(8, h, 32, dtype=torch.bfloat16, device=DEV, requires_grad=True) for h in (4, 2))
    dq, dk = (torch.zeros_like(t) for t in (q, k))

    def step():
        a, b = fa.apply_rotary_emb(q, k, cos, sin)
        return a, b, *torch.autograd.grad((a, b), (q, k), (dq, dk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b, ga, gb = step()
    for _ in range(3):
        vals = [torch.randn(t.shape, generator=g).to(t.dtype) for t in (q, k, dq, dk)]
        with torch.no_grad():
            for t, v in zip((q, k, dq, dk), vals):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for got, v, sign in zip((a, b, ga, gb), vals, (1.0, 1.0, -1.0, -1.0)):
            check(got, v, cos, sin, place, True, torch.bfloat16, sign)


def test_layouts():
    """Rows that 16-byte loads cannot take are copied, or refused in place; heads first; rows repeated."""
    print("case rotate layouts", flush=True)
    g = torch.Generator().manual_seed(12)
    cos, sin = tables(8, 32, torch.bfloat16)
    base = torch.randn(2, 3, 8, 41, generator=g).to(torch.bfloat16)
    place = torch.arange(8).expand(2, 8)
    views = [base[..., 1:33].transpose(1, 2), base[..., :40].transpose(1, 2), base[..., :32].transpose(1, 2),
             base[:, :1, :, :32].transpose(1, 2).expand(2, 8, 5, 32), base.transpose(-1, -2)[:, :, :32].permute(0, 3, 1, 2)]
    for v in views:
        x = v.to(DEV) if v.is_contiguous() else torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device=DEV)
        if not v.is_contiguous():
            src = base.to(DEV)
            x = src.as_strided(v.shape, v.stride(), v.storage_offset())
        got = fa.apply_rotary_emb(x, None, cos, sin)
        check(got, v, cos, sin, place, True, torch.bfloat16)
        with pytest.raises(RuntimeError):
            fa.apply_rotary_emb(x, None, cos, sin, inplace=True)
    wide = torch.randn(8, 33, generator=g).to(torch.bfloat16).to(DEV)
    got = fa.apply_rotary_emb(base[0].transpose(0, 1)[..., :32].to(DEV), None, wide[:, 1:17], wide[:, 17:], rotary_interleaved=False)
    check(got, base[0].transpose(0, 1)[..., :32], wide[:, 1:17], wide[:, 17:], torch.arange(8), False, torch.bfloat16)
    assert fa.apply_rotary_emb(torch.zeros(0, 4, 32, dtype=torch.float16, device=DEV), None, cos.half(), sin.half()).shape == (0, 4, 32)
    assert fa.apply_rotary_emb(torch.zeros(2, 0, 4, 32, dtype=torch.float16, device=DEV), None, cos.half(), sin.half()).shape == (2, 0, 4, 32)


def test_graph():
    """Captured forward and backward, replayed with other inputs."""
    print("case rotate graph", flush=True)
    g = torch.Generator().manual_seed(13)
    pos = torch.zeros(6, dtype=torch.int64, device=DEV)
    q, k, dq = (torch.zeros(6, h, 64, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 4))

    def step():
        cos, sin = fa.rotary_cos_sin(pos, 64)
        a, b = fa.apply_rotary_emb(q, k, cos, sin, rotary_interleaved=False)
        back = torch.ops.fa_mi355x.rotary(dq, None, cos, sin, None, None, 0, None, False, True)[0]
        return a, b, back

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        for t in (q, k, dq):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        pos.copy_(torch.randint(0, 100000, (6,), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_refusals():
    print("case rotate refusals", flush=True)
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=DEV)  # noqa: E731
    f32, i64 = torch.float32, torch.int64
    good = dict(q=mk(2, 4, 4, 64), k=mk(2, 4, 2, 64), rotary_cos=mk(9, 16), rotary_sin=mk(9, 16))
    fa.apply_rotary_emb(**good)
    for bad in (dict(q=mk(2, 4, 4, 64, dt=f32)), dict(k=mk(2, 4, 2, 64, dt=torch.float16)), dict(k=mk(2, 3, 2, 64)), dict(k=mk(2, 4, 2, 32)),
                dict(q=mk(4, 64), k=None), dict(rotary_cos=mk(9, 8)), dict(rotary_sin=mk(8, 16)), dict(rotary_cos=mk(9, 16, dt=torch.float16),
                rotary_sin=mk(9, 16, dt=torch.float16)), dict(rotary_cos=mk(9, 40), rotary_sin=mk(9, 40)), dict(rotary_cos=mk(9, 12), rotary_sin=mk(9, 12)),
                dict(rotary_cos=mk(0, 16), rotary_sin=mk(0, 16)), dict(q=mk(2, 4, 4, 60), k=None), dict(positions=mk(2, 4, dt=f32)),
                dict(positions=mk(2, 5, dt=i64)), dict(positions=mk(2, 4, dt=i64), seqlen_offsets=3), dict(positions=mk(2, 4, dt=i64).cpu()),
                dict(seqlen_offsets=mk(3, dt=torch.int32)), dict(seqlen_offsets=mk(2, dt=i64)), dict(cu_seqlens=mk(3, dt=torch.int32)),
                dict(q=mk(4, 4, 64), k=None, cu_seqlens=mk(3, dt=i64)), dict(q=mk(4, 4, 64), k=None, cu_seqlens=mk(1, dt=torch.int32)),
                dict(rotary_cos=good["rotary_cos"].cpu())):
        with pytest.raises(RuntimeError):
            fa.apply_rotary_emb(**dict(good, **bad))
    pos = mk(4, dt=i64)
    for bad in (dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=272), dict(base=0.0), dict(base=math.nan), dict(scaling="other"),
                dict(scaling="linear", factor=0.0), dict(scaling="by_parts", factor=2.0), dict(scaling="by_parts", original_length=5, low=2.0, high=2.0),
                dict(dtype=torch.float64), dict(positions=mk(4, dt=f32)), dict(positions=mk(2, 2, dt=i64)), dict(positions=pos.cpu()),
                dict(attention_factor=math.inf),
                dict(scaling="linear", factor=5e-324, base=1e-300)):
        with pytest.raises(RuntimeError):
            fa.rotary_cos_sin(**dict(dict(positions=pos, rotary_dim=32), **bad))


def test_memory_given_twice_is_not_turned_in_place():
    """Rows that share memory by any strides, and one tensor as q and as k, are refused; what lies between other rows is not."""
    x = torch.randn(4096, device=DEV).to(torch.bfloat16)
    cos, sin = fa.rotary_cos_sin(torch.arange(8, device=DEV), 32, dtype=torch.bfloat16)
    for size, stride in (((1, 4, 2, 64), (0, 64, 64, 1)), ((1, 4, 2, 64), (0, 128, 56, 1)), ((2, 3, 2, 64), (256, 128, 64, 1))):
        with pytest.raises(RuntimeError, match="repeat rows"):
            fa.apply_rotary_emb(torch.as_strided(x, size, stride), None, cos, sin, inplace=True)
    q = torch.as_strided(x, (1, 4, 2, 64), (0, 128, 64, 1))
    with pytest.raises(RuntimeError, match="same memory"):
        fa.apply_rotary_emb(q, q, cos, sin, inplace=True)
    both = x[:1536].view(1, 4, 6, 64)
    want = [t.clone() for t in fa.apply_rotary_emb(both[:, :, :4], both[:, :, 4:5], cos, sin)] + [both[:, :, 5:].clone()]
    fa.apply_rotary_emb(both[:, :, :4], both[:, :, 4:5], cos, sin, inplace=True)  # heads of one projection
    for got, t in zip((both[:, :, :4], both[:, :, 4:5], both[:, :, 5:]), want):
        assert torch.equal(got, t)
    fa.apply_rotary_emb(both.transpose(1, 2), None, cos, sin, inplace=True)  # (heads first)
