"""Calls that go through the kernels in several launches, by their tiles and heads rather than by their batch."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import capi
from oracle import fa_quant_oracle as qo
from tests.test_quant_host import FWD

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 256])
def test_many_heads(D):
    """65535 heads of 70 (or 20) sequences: the merge of what waves share would need 2^32 threads and more. All heads have
    the same rows, so all results are one result."""
    print(f"case batch parts {D}", flush=True)
    g = torch.Generator().manual_seed(91)
    B, H, keys = (70, 65535, 200) if D == 16 else (20, 65535, 100)
    k, v = (torch.randint(-127, 128, (1, 208, 1, D), generator=g).to(torch.int8) for _ in range(2))
    s = torch.full((1, 13, 1), 0.01)
    q = torch.randn(1, 1, 1, D, generator=g).to(torch.bfloat16)
    wide = lambda x: x.to(DEV).expand(-1, -1, H, *x.shape[3:])  # noqa: E731
    out, lse = fa.flash_attn_with_quantized_kvcache(
        q.to(DEV).expand(B, 1, H, D), wide(k), wide(v), wide(s), wide(s), torch.full((B,), keys, **I32),
        page_table=torch.zeros(B, 1, **I32), return_softmax_lse=True)
    rows = lambda x: qo.rows_of(x, s, [0], keys)[0]  # noqa: E731
    ref, ref_lse = qo.attend(q[0], rows(k), rows(v), torch.ones(keys, dtype=torch.bool), D ** -0.5)
    # weights (2^-11) of |v| < 1.27 and the result (2^-9) rounded, twice that
    for b in range(0, B, 5):
        assert ((out[b, 0].double() - ref[0, 0].to(DEV)).abs() <= 2 * 1.27 * (2.0 ** -11 + 2.0 ** -9)).all(), b
        assert ((lse[b, :, 0].double() - ref_lse[0, 0].item()).abs() <= 2.0 ** -16).all(), b


@pytest.mark.parametrize("heads,pages,fits", [(64, 1 << 24, True), (63, 1 << 24, True), (65, 1 << 24, False), (65, 1 << 23, True),
                                              (65535, 1 << 13, True), (65535, 1 << 15, False)])
def test_tiles_of_a_sequence(heads, pages, fits):
    """A list of tiles counts in 32 bits: 2^30 keys are 2^25 tiles of 32 for each 4, 2 or 1 heads."""
    p = capi.new_quant_fwd_params(**dict(FWD, nheads=heads, nheads_k=heads, max_pages=pages, page_table_row_stride=pages))
    assert capi.quant_fwd_workspace_size(p)[0] == (capi.FA_OK if fits else capi.FA_EINVAL), capi.last_error()
    if not fits:
        assert "heads and tokens" in capi.last_error()
