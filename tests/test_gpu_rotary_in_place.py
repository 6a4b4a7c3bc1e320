"""apply_rotary_emb in place beside autograd: gradients, and refusals that leave the rows as they were."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_rotary_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, S, D, RD = 2, 8, 64, 32


def tables():
    cos, sin = ro.table(range(S), RD)
    return cos.float().to(DEV), sin.float().to(DEV)


def rows(g, heads, **kw):
    return torch.randn(B, S, heads, D, generator=g).to(torch.bfloat16).to(DEV).requires_grad_(kw.get("requires_grad", False))


def back(d, cos, sin):
    """The gradient: turned back by the operator out of place, which test_gpu_rotary.py holds against the formula."""
    return torch.ops.fa_mi355x.rotary(d.contiguous(), None, cos, sin, None, None, 0, None, True, True)[0]


@pytest.mark.parametrize("parts", [False, True])
@pytest.mark.parametrize("need", ["both", "q", "k"])
def test_gradients(parts, need):
    """Of q and k, each a tensor of its own or a part of one projection: the bits of the operator turned back."""
    print(f"case in place gradients {parts} {need}", flush=True)
    g = torch.Generator().manual_seed(1)
    cos, sin = tables()
    d = rows(g, 6)
    x = rows(g, 6, requires_grad=need == "both" or parts)
    y = rows(g, 6, requires_grad=need == "both")
    if parts:
        both = x * 1
        q, k = both[:, :, :4], both[:, :, 4:5]
        q, k = (q, k) if need == "both" else (q, y[:, :, 4:5].detach().clone()) if need == "q" else (y[:, :, :4].detach().clone(), k)
    else:
        q, k = ((t * 1).detach().requires_grad_(n) * 1 for t, n in ((x[:, :, :4], need != "k"), (x[:, :, 4:5], need != "q")))
    plain = [t.detach().clone() for t in (q, k)]
    leaves = None if parts else [t.grad_fn.next_functions[0][0].variable if t.requires_grad else None for t in (q, k)]
    a, b = fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
    assert a is q and b is k
    want = fa.apply_rotary_emb(*plain, cos, sin)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    if not parts:
        outs = [(t, leaf, dd) for t, leaf, dd in zip((q, k), leaves, (d[:, :, :4], d[:, :, 4:5])) if leaf is not None]
        got = torch.autograd.grad([o[0] for o in outs], [o[1] for o in outs], [o[2] for o in outs])
        for gr, o in zip(got, outs):
            assert torch.equal(gr, back(o[2], cos, sin))
        return
    # the projection's own gradient, and the parts'
    ref = d.clone()
    if need != "k":
        ref[:, :, :4] = back(d[:, :, :4], cos, sin)
    if need != "q":
        ref[:, :, 4:5] = back(d[:, :, 4:5], cos, sin)
    (whole,) = torch.autograd.grad(both, x, d, retain_graph=True)
    assert torch.equal(whole, ref)
    turned = [(t, s) for t, s, n in ((q, slice(0, 4), need != "k"), (k, slice(4, 5), need != "q")) if n]
    (of_parts,) = torch.autograd.grad([t for t, _ in turned], x, [d[:, :, s] for _, s in turned])
    for _, s in turned:
        assert torch.equal(of_parts[:, :, s], ref[:, :, s])


def test_twice_and_second_gradients():
    print("case in place twice", flush=True)
    g = torch.Generator().manual_seed(2)
    cos, sin = tables()
    x, d, w = rows(g, 3, requires_grad=True), rows(g, 3, requires_grad=True), rows(g, 3)
    q = x * 1
    fa.apply_rotary_emb(q, None, cos, sin, inplace=True)
    fa.apply_rotary_emb(q, None, cos, sin, inplace=True)
    (first,) = torch.autograd.grad(q, x, d, create_graph=True)
    assert torch.equal(first, back(back(d.detach(), cos, sin), cos, sin))
    (second,) = torch.autograd.grad(first, d, w)
    once = fa.apply_rotary_emb(w, None, cos, sin)
    assert torch.equal(second, fa.apply_rotary_emb(once, None, cos, sin))


def test_refusals_leave_the_rows():
    """What autograd does not let be changed is refused with its rows as they were, and an argument that is refused leaves
    no history."""
    print("case in place refusals", flush=True)
    g = torch.Generator().manual_seed(3)
    cos, sin = tables()
    leaf = rows(g, 4, requires_grad=True)
    pieces = (rows(g, 4, requires_grad=True) * 1).split(2, 2)
    for q, k in ((leaf, None), (leaf[:, :, 1:], None), (pieces[0], None), (pieces[0], pieces[1]), (rows(g, 4, requires_grad=True) * 1, leaf)):
        given = [t for t in (q, k) if t is not None]
        before = [(t.detach().clone(), t._version, t.grad_fn) for t in given]
        with pytest.raises(RuntimeError):
            fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
        for t, (bits, version, fn) in zip(given, before):
            assert torch.equal(t, bits) and t._version == version and t.grad_fn is fn
    q = rows(g, 4, requires_grad=True) * 1
    bits, fn = q.detach().clone(), q.grad_fn
    for bad in (dict(rotary_cos=cos[:, :12], rotary_sin=sin[:, :12]), dict(positions=torch.zeros(B, S + 1, dtype=torch.int64, device=DEV)), dict(k=q)):
        with pytest.raises(RuntimeError):
            fa.apply_rotary_emb(**dict(dict(q=q, k=None, rotary_cos=cos, rotary_sin=sin, inplace=True), **bad))
        assert torch.equal(q, bits) and q.grad_fn is fn


def test_saved_rows_are_missed():
    """The case that gave wrong gradients: a factor turned after it was saved."""
    print("case in place saved", flush=True)
    g = torch.Generator().manual_seed(4)
    cos, sin = tables()
    x, w = rows(g, 4), rows(g, 4, requires_grad=True)
    y = (x * w).sum()
    fa.apply_rotary_emb(x, None, cos, sin, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("inplace", [False, True])
def test_compiled(inplace):
    """A step with the rotation, traced: eager results."""
    print(f"case in place compiled {inplace}", flush=True)
    g = torch.Generator().manual_seed(5)
    cos, sin = tables()
    x, d = rows(g, 4, requires_grad=True), rows(g, 4)

    def step(x):
        q = fa.apply_rotary_emb(x * 2, None, cos, sin, inplace=inplace)
        return q * 0.5

    want = step(x)
    (grad,) = torch.autograd.grad(want, x, d)
    got = torch.compile(step, backend="aot_eager")(x)
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, x, d)[0], grad)


def test_memory_in_common():
    """q and k of one projection, side by side or alternating by heads, are turned; a head that both hold is refused."""
    print("case in place common memory", flush=True)
    g = torch.Generator().manual_seed(6)
    cos, sin = tables()
    base = rows(g, 9)
    alternate = base.view(B, S, 3, 3, D)
    for q, k in ((base[:, :, 2:6], base[:, :, :2]), (alternate[:, :, :, 0], alternate[:, :, :, 1]), (base[:, :4, :4], base[:, 4:, 3:5]),
                 (base[:, ::2, :4], base[:, 1::2, 3:5]), (base[0, :, :4][None], base[1, :, 3:5][None])):
        want = [t.clone() for t in fa.apply_rotary_emb(q, k, cos, sin)]
        rest = base.clone()
        fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        q.zero_(), k.zero_()
        turned = base != rest  # zeros where q and k are; the rest as it was
        assert (base[turned] == 0).all() and turned.sum() <= q.numel() + k.numel()
        base.copy_(rest)
    before = base.clone()
    for q, k in ((base[:, :, :4], base[:, :, 3:5]), (base[:, :, 3:5], base[:, :, :4]), (base[:, :, :4], base[:, :, :4]),
                 (alternate[:, :, :, 0], base[:, :, 3:4]), (base[0, :, :4][None], base[0, :, 2:3][None])):
        with pytest.raises(RuntimeError, match="same memory"):
            fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
    assert torch.equal(base, before)


def test_farthest_offsets():
    """Rows whose place in the tables passes 64 bits take the nearest row like others outside."""
    print("case rotate farthest offsets", flush=True)
    g = torch.Generator().manual_seed(7)
    cos, sin = tables()
    q = rows(g, 2)
    for offset, row in ((2 ** 63 - 1, S - 1), (2 ** 63 - 4, S - 1), (-2 ** 63, 0), (2 ** 31, S - 1), (-2 ** 31, 0)):
        at = torch.full((B, S), row, dtype=torch.int32, device=DEV)
        assert torch.equal(fa.apply_rotary_emb(q, None, cos, sin, seqlen_offsets=offset), fa.apply_rotary_emb(q, None, cos, sin, positions=at)), offset


@pytest.mark.parametrize("inplace", [False, True])
def test_traced_and_transformed_backward(inplace):
    """Compiled autograd and torch.func.grad (in place; out of place it is refused): the eager gradient."""
    print(f"case in place traced backward {inplace}", flush=True)
    import torch._dynamo.compiled_autograd as compiled

    g = torch.Generator().manual_seed(8)
    cos, sin = tables()
    d = rows(g, 5)
    pos = torch.randint(0, S, (B, S), generator=g).to(DEV)

    def loss(x):
        both = x * 1
        q, k = fa.apply_rotary_emb(both[:, :, :4], both[:, :, 4:], cos, sin, positions=pos, inplace=inplace)
        return (q * d[:, :, :4]).sum() + (k * d[:, :, 4:]).sum()

    x = rows(g, 5, requires_grad=True)
    (want,) = torch.autograd.grad(loss(x), x)
    value = loss(x)
    with compiled._enable(lambda gm: torch.compile(gm, backend="eager")):
        value.backward()
    assert torch.equal(x.grad, want)
    if inplace:
        assert torch.equal(torch.func.grad(loss)(x.detach()), want)
    else:
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.grad(loss)(x.detach())


@pytest.mark.parametrize("grad", [False, True])
def test_captured(grad):
    """A step that turns parts of a projection in place, captured and replayed with other values; on a stream of its own before."""
    print(f"case in place captured {grad}", flush=True)
    g = torch.Generator().manual_seed(9)
    cos, sin = tables()
    x, d = rows(g, 6, requires_grad=grad), rows(g, 6)
    pos = torch.zeros(B, S, dtype=torch.int64, device=DEV)

    def step():
        both = x * 1
        fa.apply_rotary_emb(both[:, :, :4], both[:, :, 4:5], cos, sin, positions=pos, inplace=True)
        # (no step's history may outlive it: a backward pass of the same leaf cannot be captured beside one)
        return (both.detach(), *torch.autograd.grad(both, x, d)) if grad else (both,)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            early = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(early, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        with torch.no_grad():
            for t in (x, d):
                t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        pos.copy_(torch.randint(0, S, pos.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_no_rows_and_one():
    print("case in place sizes", flush=True)
    cos, sin = tables()
    for shape in ((0, 4, 3, D), (2, 0, 3, D), (0, 3, D), (1, 1, 1, D), (1, 1, D)):
        x = torch.ones(shape, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        q, k = x * 1, x.detach()[..., :1, :].clone()
        before = q.detach().clone(), k.clone()
        a, b = fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
        want = fa.apply_rotary_emb(*before, cos, sin)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
        (gr,) = torch.autograd.grad(a, x, torch.ones_like(a))
        assert gr.shape == x.shape
