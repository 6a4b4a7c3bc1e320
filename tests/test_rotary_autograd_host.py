"""What autograd is told of the rotation, on meta tensors: versions of what is turned in place."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import ops

META = dict(device="meta")


def tables():
    return torch.empty(9, 16, **META), torch.empty(9, 16, **META)


def rows(heads=4, **kw):
    return torch.empty(2, 5, heads, 64, dtype=torch.bfloat16, **META, **kw)


@pytest.mark.parametrize("with_k", [True, False])
def test_in_place_raises_the_version(with_k):
    cos, sin = tables()
    q, k = rows(), rows(2) if with_k else None
    given = [t for t in (q, k, cos, sin) if t is not None]
    for call in (lambda: fa.apply_rotary_emb(q, k, cos, sin, inplace=True),
                 lambda: ops.rotary_(q, k, cos, sin, None, None, 0, None, True, False)):
        before = [t._version for t in given]
        call()
        turned = 2 if with_k else 1
        assert all(t._version > b for t, b in zip(given[:turned], before))
        assert [t._version for t in given[turned:]] == before[turned:]
    before = q._version
    with torch.no_grad():
        fa.apply_rotary_emb(q[:, :, 1:], None, cos, sin, inplace=True)  # a part has its tensor's version
    assert q._version > before
    before = q._version
    with torch.inference_mode():
        fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
    assert q._version > before


def test_saved_before_it_is_turned():
    """Backward of a product whose factor was turned in place after: autograd refuses, as for any other change."""
    cos, sin = tables()
    for q_needs in (False, True):
        q, w = rows(requires_grad=q_needs), rows(requires_grad=True)
        y = (q * w).sum()
        with torch.no_grad():
            fa.apply_rotary_emb(q, None, cos, sin, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_inference_tensors_stay_in_inference():
    """As for torch's own operations in place: refused outside of inference_mode, allowed in it."""
    cos, sin = tables()
    with torch.inference_mode():
        q = rows()
        fa.apply_rotary_emb(q, None, cos, sin, inplace=True)
    with pytest.raises(RuntimeError, match="(?i)inference"):
        fa.apply_rotary_emb(q, None, cos, sin, inplace=True)


def refused_in_place():
    """Rows that autograd does not let be changed, by what makes them so."""
    leaf = rows(requires_grad=True)
    yield "a leaf", leaf, None
    yield "a part of a leaf", leaf[:, :, 1:], None
    yield "pieces of one call", (rows(requires_grad=True) * 1).split(2, 2)[0], None
    yield "pieces of one call, as k", rows(requires_grad=True) * 1, (rows(requires_grad=True) * 1).unbind(0)[0][None].expand(2, 5, 4, 64)
    yield "k a leaf", rows(requires_grad=True) * 1, leaf
    with torch.no_grad():
        part = leaf[:, :, 1:]
    yield "a part taken without gradients", part, None


@pytest.mark.parametrize("direct", [False, True])
def test_refused_before_anything_is_turned(direct):
    cos, sin = tables()
    for why, q, k in refused_in_place():
        given = [t for t in (q, k) if t is not None]
        before = [(t._version, t.grad_fn) for t in given]
        with pytest.raises(RuntimeError):
            if direct:
                ops.rotary_(q, k, cos, sin, None, None, 0, None, True, False)
            else:
                fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
        assert [t._version for t in given] == [b[0] for b in before], why
        assert all(t.grad_fn is b[1] for t, b in zip(given, before)), why
    with torch.inference_mode():
        cos, sin = tables()
    q = rows(requires_grad=True) * 1
    before = q._version
    with pytest.raises(RuntimeError, match="(?i)inference tensors"):  # they cannot be kept for the backward pass
        fa.apply_rotary_emb(q, None, cos, sin, inplace=True)
    assert q._version == before


def test_history_in_place():
    """Whoever needs a gradient gets the turn's history, and nothing else does."""
    cos, sin = tables()
    for need_q, need_k in ((True, True), (True, False), (False, True), (False, False)):
        x, y = rows(requires_grad=need_q), rows(2, requires_grad=need_k)
        q, k = x * 1, y * 1
        a, b = fa.apply_rotary_emb(q, k, cos, sin, inplace=True)
        assert a is q and b is k and (q.requires_grad, k.requires_grad) == (need_q, need_k)
        if need_q or need_k:
            (a.sum() + b.sum()).backward()
        assert (x.grad is not None, y.grad is not None) == (need_q, need_k)
    q = rows(requires_grad=True) * 1
    with torch.no_grad():
        fa.apply_rotary_emb(q, None, cos, sin, inplace=True)
    assert "Mul" in type(q.grad_fn).__name__


def test_tables_changed_before_the_backward_pass():
    cos, sin = tables()
    for inplace in (False, True):
        q = rows(requires_grad=True) * 1
        out = fa.apply_rotary_emb(q, None, cos, sin, inplace=inplace)
        cos.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


@pytest.mark.parametrize("inplace", [False, True])
def test_no_forward_mode(inplace):
    """Tangents of rows or of tables are refused, not dropped; the rows then are as they were."""
    fw = torch.autograd.forward_ad
    for of in ("q", "k", "cos", "sin"):
        for needs in (False, True):
            with fw.dual_level():
                cos, sin = tables()
                args = dict(q=rows(), k=rows(2), cos=cos, sin=sin)
                plain = args[of].clone()
                args[of] = fw.make_dual(plain.requires_grad_() * 1 if needs and of in "qk" else plain, torch.empty_like(plain))
                before = [t._version for t in args.values()]
                with pytest.raises(RuntimeError, match="forward"):
                    fa.apply_rotary_emb(*args.values(), inplace=inplace)
                assert [t._version for t in args.values()] == before
    cos, sin = tables()
    with pytest.raises(RuntimeError, match="forward"):
        torch.func.jvp(lambda q: fa.apply_rotary_emb(q, None, cos, sin, inplace=inplace), (rows(),), (rows(),))
    with fw.dual_level(), torch.no_grad():
        q = fw.make_dual(rows(), rows())
        with pytest.raises(RuntimeError, match="forward"):
            ops.rotary_(q, None, cos, sin, None, None, 0, None, True, False)
        fa.apply_rotary_emb(rows(), None, cos, sin, inplace=inplace)  # none of its own


@pytest.mark.parametrize("with_k", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_compiled_autograd(inplace, with_k):
    """The backward pass traced by torch's compiled autograd."""
    import torch._dynamo.compiled_autograd as compiled

    cos, sin = tables()
    x, y = rows(requires_grad=True), rows(2, requires_grad=True) if with_k else None
    out = fa.apply_rotary_emb(x * 1, y * 1 if with_k else None, cos, sin, inplace=inplace)
    with compiled._enable(lambda gm: torch.compile(gm, backend="eager")):
        (out[0].sum() + out[1].sum() if with_k else out.sum()).backward()
    assert x.grad.shape == x.shape and (y is None or y.grad.shape == y.shape)
