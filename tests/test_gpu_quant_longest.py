"""The longest sequence that attention over 8-bit codes takes, 2^30 tokens, with windows as wide as they come."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import capi
from tests.test_quant_host import FWD

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("right", [2 ** 31 - 1, 2 ** 30, 2 ** 30 - 1, 5, -1])
@pytest.mark.parametrize("sq", [1, 3, 40])
def test_right_window_at_the_end(sq, right):
    """1024 pages of 2^20 tokens, all of them one page but the last; the left window leaves the last 8 keys to each row."""
    print(f"case longest {sq} {right}", flush=True)
    g = torch.Generator().manual_seed(71)
    P, D = 1 << 20, 16
    k = torch.zeros(2, P, 1, D, dtype=torch.int8, device=DEV)
    v = torch.zeros(2, P, 1, D, dtype=torch.int8, device=DEV)
    tail = torch.randint(-127, 128, (64, D), generator=g).to(torch.int8)
    v[1, -64:, 0] = tail.to(DEV)
    s = torch.full((2, 1, 1), 0.02, device=DEV)
    table = torch.zeros(1, 1024, **I32)
    table[0, -1] = 1
    q = torch.randn(1, sq, 1, D, generator=g).to(torch.float16)
    out, lse = fa.flash_attn_with_quantized_kvcache(q.to(DEV), k, v, s, s, torch.tensor([1 << 30], **I32), page_table=table,
                                                    window_size=(7, right), return_softmax_lse=True)
    for r in range(sq):  # scores are 0: the mean of the keys that the row sees
        i = 63 - (sq - 1 - r)
        seen = tail[i - 7:(64 if right < 0 else min(64, i + right + 1))].double() * 0.02
        want = seen.mean(0)
        # weights that are powers of two of each other, sums of 64 terms, the result rounded to fp16
        assert ((out[0, r, 0].cpu().double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -11 * 127 * 0.02 + 2.0 ** -24).all()
        assert abs(lse[0, 0, r].item() - torch.tensor(float(len(seen))).log().item()) <= 2.0 ** -20


@pytest.mark.parametrize("rows,fits", [(1 << 27, True), ((1 << 27) + 1, False)])
def test_query_rows(rows, fits):
    """Positions of rows count down from 0 where there are more of them than keys: 2^30 packed rows at most (here 2 x 4
    of each)."""
    p = capi.new_quant_fwd_params(**dict(FWD, seqlen_q=rows))
    assert capi.quant_fwd_workspace_size(p)[0] == (capi.FA_OK if fits else capi.FA_EINVAL)
    if not fits:
        assert "too many query rows" in capi.last_error()
