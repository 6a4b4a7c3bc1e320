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
